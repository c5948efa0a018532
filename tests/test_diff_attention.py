"""Differential attention (vit_amd.diff_attention): forward and gradients against the formula in 64 bits with element-wise
bounds, gradients against differences, masks and rows without keys, layouts, capture, refusals.

Bounds.  u is the half step of the operands' rounding (2^-8 bf16, nothing for f32) plus what f32 arithmetic adds to a
probability: roundings of d products in a score of size smax and of nk additions in a denominator, taken as independent
(their square roots, with a factor of 8 and 4), and the exponential's."""
import math

import pytest
import torch

import vit_amd
from vit_amd import VitkError, lib

gpu = pytest.mark.gpu
F, H16 = torch.float32, torch.bfloat16


def _inputs(B, nq, nk, H, K, d, dtype, lens=None, shared=False, seed=0):
    g = torch.Generator().manual_seed(seed + nq * 7 + nk)
    rnd = lambda *s: torch.randn(*s, generator=g)                              # noqa: E731
    q, k = rnd(B, nq, H, 2, d).to(dtype), rnd(B, nk, K, 2, d).to(dtype)
    v, do = rnd(B, nk, K, 2 * d).to(dtype), rnd(B, nq, H, 2 * d).to(dtype)
    lam = rnd(*((4, d) if shared else (4, H, d))) * (1.2 / d ** 0.5)
    kl = None if lens is None else torch.tensor(lens, dtype=torch.int32)
    return q, k, v, lam, do, kl


def reference(q, k, v, lam, do, kl, lambda_init, scale, causal, dtype):
    """{name: (value, bound)} in 64 bits, on the GPU (a fast place for double products)."""
    q, k, v, lam, do = (t.double().cuda() for t in (q, k, v, lam, do))
    B, nq, H, _, d = q.shape
    nk, K = k.shape[1], k.shape[2]
    g = H // K
    seen = torch.ones(B, 1, nq, nk, dtype=torch.bool, device="cuda")
    if kl is not None:
        seen = seen & (torch.arange(nk, device="cuda") < kl.cuda()[:, None, None, None])
    if causal:
        seen = seen & torch.ones(nq, nk, dtype=torch.bool, device="cuda").tril(nk - nq)
    hidden = ~(torch.arange(nk, device="cuda") < (kl.cuda()[:, None] if kl is not None else nk)).expand(B, nk)
    k = k.masked_fill(hidden[:, :, None, None, None], 0.0)
    v = v.masked_fill(hidden[:, :, None, None], 0.0)
    Q = q.permute(3, 0, 2, 1, 4)                                               # [2, B, H, nq, d]
    KK = k.permute(3, 0, 2, 1, 4).repeat_interleave(g, 2)
    V = v.permute(0, 2, 1, 3).repeat_interleave(g, 1)
    DO = do.permute(0, 2, 1, 3)
    s = (Q @ KK.transpose(-1, -2)) * scale
    smax = float(((Q.abs() @ KK.abs().transpose(-1, -2)) * scale).max())
    p = s.masked_fill(~seen, -math.inf).softmax(-1).nan_to_num(0.0)
    L = (lam if lam.dim() == 3 else lam[:, None].expand(4, H, d))
    e1, e2 = (L[0] * L[1]).sum(-1).exp(), (L[2] * L[3]).sum(-1).exp()
    w = (e1 - e2 + lambda_init).view(1, H, 1, 1)
    r32 = 2.0 ** -24 * (8 * math.sqrt(d) * smax + 4 * math.sqrt(nk) + 64)      # a probability's relative error in f32
    half = 2.0 ** -8 if dtype == H16 else 2.0 ** -24
    u = r32 + (half if dtype == H16 else 0.0)
    A = p[0] - w * p[1]
    Aabs = p[0] + w.abs() * p[1]
    O, O2, M = A @ V, p[1] @ V, Aabs @ V.abs()
    ew = 2.0 ** -24 * (8 * math.sqrt(d) + 16) * (e1 * ((L[0] * L[1]).abs().sum(-1) + 1) + e2 * ((L[2] * L[3]).abs().sum(-1) + 1) + abs(lambda_init))
    EW = ew.view(1, H, 1, 1)
    out_b = u * M + half * O.abs() + EW * O2.abs()
    dA = DO @ V.transpose(-1, -2)
    eA = 2.0 ** -24 * 8 * math.sqrt(2 * d) * (DO.abs() @ V.abs().transpose(-1, -2))
    D = (p * dA).sum(-1, keepdim=True)
    # D_m comes from O and O_2, which carry the probabilities' error and their own rounding to the type
    eD = ((u * M + half * O.abs() + w.abs() * (u * (p[1] @ V.abs()) + half * O2.abs()) + EW * O2.abs()) * DO.abs()).sum(-1, keepdim=True)
    eD = eD * 1.01 + 2.0 ** -24 * 8 * math.sqrt(2 * d) * (DO.abs() * (O.abs() + w.abs() * O2.abs())).sum(-1, keepdim=True)
    c = torch.stack([torch.ones_like(w), -w])
    dS = c * p * (dA - D)
    edS = u * dS.abs() + c.abs() * p * (eA + eD + r32 * (dA - D).abs()) + EW * p * (dA - D).abs()
    head = lambda t: t.permute(0, 2, 1, 3)                                     # noqa: E731
    fold = lambda t: t.unflatten(1, (K, g)).sum(2)                             # noqa: E731
    res = {"out": (head(O), head(out_b))}
    dq, edq = dS @ KK * scale, edS @ KK.abs() * scale
    res["dq"] = tuple(t.permute(1, 3, 2, 0, 4) for t in (dq, edq * 1.01 + half * dq.abs()))
    dk = torch.stack([fold(dS[m].transpose(-1, -2) @ Q[m]) for m in (0, 1)]) * scale
    edk = torch.stack([fold(edS[m].transpose(-1, -2) @ Q[m].abs()) for m in (0, 1)]) * scale
    res["dk"] = tuple(t.permute(1, 3, 2, 0, 4) for t in (dk, edk * 1.01 + half * dk.abs() + 2.0 ** -20 * edk))
    dv = fold(A.transpose(-1, -2) @ DO)
    # the maps' probabilities meet dO apart, each rounded to the type: u P_1 + u |w| P_2
    edv = fold((u * Aabs + EW * p[1]).transpose(-1, -2) @ DO.abs())
    res["dv"] = tuple(head(t) for t in (dv, edv * 1.01 + half * dv.abs()))
    dw = -(p[1] * dA).sum((0, 2, 3))
    edw = (p[1] * (r32 * dA.abs() + eA)).sum((0, 2, 3))                        # f32 in both types
    dl = torch.stack([dw[:, None] * e1[:, None] * L[1], dw[:, None] * e1[:, None] * L[0],
                      -dw[:, None] * e2[:, None] * L[3], -dw[:, None] * e2[:, None] * L[2]])
    rel_e = 2.0 ** -24 * (8 * math.sqrt(d) * 4 + 64)
    edl = torch.stack([edw[:, None] * e1[:, None] * L[1].abs(), edw[:, None] * e1[:, None] * L[0].abs(),
                       edw[:, None] * e2[:, None] * L[3].abs(), edw[:, None] * e2[:, None] * L[2].abs()]) + rel_e * dl.abs()
    if lam.dim() == 2:
        dl, edl = dl.sum(1), edl.sum(1)
    res["dlam"] = (dl, edl)
    return res


def _check(got, want, name):
    value, bound = want
    got = got.double()
    assert got.shape == value.shape
    assert got.isfinite().all(), name
    err = (got - value).abs()
    bad = err > bound + 1e-30
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} values, worst {float((err / (bound + 1e-30)).max()):.2f} of the bound"


def _run(case, dtype, lens=None, causal=False, shared=False, lambda_init=0.6, scale=None, backward=True):
    q, k, v, lam, do, kl = _inputs(*case, dtype, lens, shared)
    sc = case[-1] ** -0.5 if scale is None else scale
    want = reference(q, k, v, lam, do, kl, lambda_init, sc, causal, dtype)
    leaves = [t.cuda().requires_grad_(backward) for t in (q, k, v, lam)]
    out = vit_amd.diff_attention(*leaves, lambda_init, scale=scale, key_lens=None if kl is None else kl.cuda(), causal=causal)
    assert out.dtype == dtype
    _check(out.detach(), want["out"], "out")
    if backward:
        for n, t in zip(("dq", "dk", "dv", "dlam"), torch.autograd.grad(out, leaves, do.cuda())):
            _check(t, want[n], n)


#        B, nq, nk, H, K, d
CASES = [
    ((1, 1, 1, 1, 1, 8), {}),
    ((2, 1, 5, 2, 1, 16), {}),
    ((3, 1, 2100, 8, 2, 64), dict(lens=[2100, 1, 777])),                        # one token, split keys, shared heads
    ((1, 1, 9001, 4, 4, 32), dict(shared=True)),
    ((2, 7, 333, 6, 2, 40), dict(causal=True)),                                 # a few tokens behind a cache
    ((2, 5, 300, 10, 2, 24), dict(causal=True, lens=[300, 290])),               # rows of several heads in one tile
    ((2, 197, 197, 12, 12, 32), dict(shared=True)),
    ((1, 577, 577, 2, 2, 48), {}),
    ((2, 129, 129, 3, 3, 64), dict(causal=True)),
    ((1, 300, 300, 4, 2, 64), dict(causal=True, lens=[123])),
    ((4, 50, 70, 4, 4, 24), dict(lens=[0, 70, 1, 33])),                         # an empty sample
    ((1, 90, 40, 2, 2, 32), dict(causal=True)),                                 # the first 50 queries see nothing
    ((16, 197, 197, 4, 4, 32), {}),                                             # many rows: 128 to a workgroup from here on
    ((64, 40, 50, 4, 2, 56), dict(lens=[(7 * i) % 51 for i in range(64)])),
    ((4, 513, 513, 8, 4, 64), dict(causal=True)),
    ((33, 65, 33, 4, 4, 48), dict(causal=True, lens=[33 - i for i in range(33)])),
    ((130, 31, 64, 1, 1, 8), dict(shared=True)),
    ((3, 1000, 777, 45, 45, 16), {}),
]


@gpu
@pytest.mark.parametrize("dtype", [H16, F])
@pytest.mark.parametrize("case,kw", CASES)
def test_forward_and_gradients(case, kw, dtype):
    _run(case, dtype, **kw)


@gpu
@pytest.mark.parametrize("dtype", [H16, F])
@pytest.mark.parametrize("d", [8, 16, 24, 32, 40, 48, 56, 64])
def test_every_head_size(d, dtype):
    _run((2, 70, 95, 4, 2, d), dtype)
    _run((70, 70, 95, 4, 2, d), dtype, backward=False)


SPLIT = [                                                                       # the backward's parts, added by kernels of their own
    ((2, 40, 1500, 4, 2, 40), dict(causal=True, lens=[1500, 700])),             # keys split, the second sample's in part
    ((1, 600, 600, 2, 1, 48), dict(causal=True)),                               # rows and keys split
    ((1, 1030, 1030, 4, 1, 64), dict(causal=True, shared=True)),
    ((2, 700, 530, 3, 1, 16), dict(lens=[0, 530])),                             # an empty sample, a group of three
    ((1, 5, 2570, 5, 1, 8), {}),
    ((1, 1100, 1050, 9, 9, 24), dict(causal=True)),                             # f32 in parts, bf16 not
]


@gpu
@pytest.mark.parametrize("dtype", [H16, F])
@pytest.mark.parametrize("case,kw", SPLIT)
def test_gradients_in_parts(case, kw, dtype):
    _run(case, dtype, **kw)


@gpu
@pytest.mark.parametrize("dtype", [H16, F])
def test_other_scales_and_weights(dtype):
    _run((2, 40, 60, 2, 2, 32), dtype, scale=0.02, lambda_init=0.0)
    _run((2, 40, 60, 2, 2, 32), dtype, scale=1.5, lambda_init=-3.0)
    _run((2, 40, 60, 6, 2, 48), dtype, lambda_init=-3.0)                        # negative and shared
    _run((2, 40, 60, 6, 2, 64), dtype, lambda_init=-0.3)                        # of both signs in a group


@gpu
def test_gradients_against_differences():
    q, k, v, lam, do, _ = _inputs(2, 9, 14, 4, 2, 16, F)
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v, lam)]
    got = torch.autograd.grad(vit_amd.diff_attention(*leaves, 0.4, causal=True), leaves, do.cuda())
    for i in range(4):
        move = torch.randn(leaves[i].shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64)

        def loss(step):
            t = [x.double() for x in (q, k, v, lam)]
            t[i] = t[i] + step * move
            return float((reference(*t, do, None, 0.4, 0.25, True, F)["out"][0].cpu() * do.double()).sum())
        want = (loss(1e-5) - loss(-1e-5)) / 2e-5
        have = float((got[i].double().cpu() * move).sum())
        assert abs(have - want) <= 1e-4 * (1 + abs(want)), (i, have, want)


@gpu
@pytest.mark.parametrize("dtype", [H16, F])
@pytest.mark.parametrize("B", [2, 70])                                          # both forms
def test_hidden_keys_are_never_read(B, dtype):
    lens = [(5 + 11 * i) % 60 for i in range(B)]
    q, k, v, lam, do, kl = _inputs(B, 66, 60, 2, 2, 32, dtype, lens)
    a = [t.cuda().requires_grad_(True) for t in (q, k, v, lam)]
    k2, v2 = k.clone(), v.clone()
    for b, n in enumerate(lens):
        k2[b, n:] = float("nan")
        v2[b, n:] = float("inf")
    c = [t.cuda().requires_grad_(True) for t in (q, k2, v2, lam)]
    x = vit_amd.diff_attention(*a, key_lens=kl.cuda())
    y = vit_amd.diff_attention(*c, key_lens=kl.cuda())
    assert torch.equal(x, y) and (x[torch.tensor(lens) == 0] == 0).all()
    for s, t in zip(torch.autograd.grad(x, a, do.cuda()), torch.autograd.grad(y, c, do.cuda())):
        assert torch.equal(s, t)
    gk = torch.autograd.grad(vit_amd.diff_attention(*c, key_lens=kl.cuda()), c[1], do.cuda())[0]
    for b, n in enumerate(lens):
        assert (gk[b, n:] == 0).all()


@gpu
def test_key_lens_outside_the_keys_are_clamped():
    q, k, v, lam, _, _ = (None if t is None else t.cuda() for t in _inputs(2, 5, 40, 2, 2, 32, H16))
    lens = torch.tensor([1000, -3], dtype=torch.int32, device="cuda")
    out = vit_amd.diff_attention(q, k, v, lam, key_lens=lens)
    assert torch.equal(out[0], vit_amd.diff_attention(q, k, v, lam)[0]) and (out[1] == 0).all()


@gpu
@pytest.mark.parametrize("dtype", [H16, F])
def test_extreme_scores_and_non_finite_rows(dtype):
    q, k, v, lam, _, _ = _inputs(1, 64, 64, 2, 2, 32, dtype)
    q = q * 100                                                               # one-hot maps
    want = reference(q, k, v, lam, torch.zeros(1, 64, 2, 64), None, 0.5, 32 ** -0.5, False, dtype)["out"][0]
    got = vit_amd.diff_attention(q.cuda(), k.cuda(), v.cuda(), lam.cuda(), 0.5)
    assert got.isfinite().all()
    # scores near 1000 carry 1000 * 8 sqrt(32) * 2^-24 = 3e-3 of absolute error into the exponent
    assert (got.double() - want).abs().max() <= 0.1
    q[0, 3, 1, 0, 5] = float("nan")
    out = vit_amd.diff_attention(q.cuda(), k.cuda(), v.cuda(), lam.cuda(), 0.5)
    assert out[0, 3, 1].isnan().all()
    out[0, 3, 1] = 0
    assert out.isfinite().all()


@gpu
@pytest.mark.parametrize("dtype", [H16, F])
def test_layouts(dtype):
    """The fused projection's head-major tensor, a token-major one, padded rows and one value for all samples."""
    B, N, H, d = 3, 77, 4, 32
    q, k, v, lam, do, _ = (None if t is None else t.cuda() for t in _inputs(B, N, N, H, H, d, dtype))
    lead = [q, k, v, lam]
    want = vit_amd.diff_attention(*[t.requires_grad_(True) for t in lead])
    grads = torch.autograd.grad(want, lead, do)

    def check(q2, k2, v2):
        ins = [q2, k2, v2, lam]
        out = vit_amd.diff_attention(*ins)
        assert torch.equal(out, want)
        for a, b in zip(torch.autograd.grad(out, ins, do), grads):
            assert torch.equal(a, b)
    with torch.no_grad():
        qkv = torch.stack([q.permute(0, 2, 1, 3, 4).reshape(B, H, N, 2 * d), k.permute(0, 2, 1, 3, 4).reshape(B, H, N, 2 * d),
                           v.permute(0, 2, 1, 3)]).contiguous()
        rows = torch.cat([q.reshape(B, N, -1), k.reshape(B, N, -1), v.reshape(B, N, -1)], -1)
        wide = torch.full((B, N + 3, H, 2, d + 8), 9.0, dtype=dtype, device="cuda")
        wide[:, :N, :, :, :d] = q
    hm = [qkv[i].view(B, H, N, 2, d).permute(0, 2, 1, 3, 4) for i in (0, 1)] + [qkv[2].permute(0, 2, 1, 3)]
    check(*[t.requires_grad_(True) for t in hm])
    D = 2 * d * H
    tm = [rows[..., :D].view(B, N, H, 2, d), rows[..., D:2 * D].view(B, N, H, 2, d), rows[..., 2 * D:].view(B, N, H, 2 * d)]
    check(*[t.requires_grad_(True) for t in tm])
    check(wide[:, :N, :, :, :d].requires_grad_(True), k, v)
    one = k.detach()[:1].expand(B, N, H, 2, d)
    a = one.clone().requires_grad_(True)
    b = k.detach()[:1].clone().requires_grad_(True)
    ga, = torch.autograd.grad(vit_amd.diff_attention(q, a, v, lam), a, do)
    gb, = torch.autograd.grad(vit_amd.diff_attention(q, b.expand(B, N, H, 2, d), v, lam), b, do)
    assert torch.allclose(gb.float(), ga.float().sum(0, keepdim=True), rtol=2 ** -6, atol=0.05 if dtype == H16 else 1e-5)


@gpu
def test_gradients_that_arrive_in_any_layout():
    """A gradient at an odd address, transposed, or broadcast: copied first, with the same values after."""
    q, k, v, lam, do, _ = _inputs(2, 40, 50, 4, 2, 16, H16)
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v, lam)]
    do = do.cuda()
    out = vit_amd.diff_attention(*leaves)
    want = torch.autograd.grad(out, leaves, do, retain_graph=True)
    odd = torch.empty(do.numel() + 1, dtype=do.dtype, device="cuda")
    odd[1:] = do.reshape(-1)
    for g in (odd[1:].view(do.shape), do.transpose(1, 2).contiguous().transpose(1, 2)):
        for a, b in zip(torch.autograd.grad(out, leaves, g, retain_graph=True), want):
            assert torch.equal(a, b)
    ones = torch.autograd.grad(out, leaves, torch.ones_like(out), retain_graph=True)
    for a, b in zip(torch.autograd.grad(out.sum(), leaves), ones):
        assert torch.equal(a, b)


@gpu
def test_learned_weight_collects_no_one_sided_error():
    """w's gradient sums -P_2 dA over 73,856 rows whose own terms cancel.  The matrix pipe's products lean to one side by some
    1e-9, which adds up to 7e-5 in the sum where every row leans alike; the backward negates every other row."""
    B, N, H, d, w0 = 16, 577, 8, 48, 0.6
    rows = B * N * H
    errors = []
    for seed in (20, 21, 22, 23):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")          # noqa: E731
        q, k, v, do = (rnd(*s).to(H16) for s in ((B, N, H, 2, d), (B, N, H, 2, d), (B, N, H, 2 * d), (B, N, H, 2 * d)))
        lam = (rnd(4, d) * 0.1).requires_grad_(True)
        dlam = torch.autograd.grad(vit_amd.diff_attention(q, k, v, lam, w0), lam, do)[0].double()
        dw = 0.0
        for b in range(B):
            Q, K = (t[b, :, :, 1].double().permute(1, 0, 2) for t in (q, k))
            p = torch.softmax(Q @ K.transpose(1, 2).contiguous() * d ** -0.5, -1)
            dw -= float(((p @ v[b].double().permute(1, 0, 2)) * do[b].double().permute(1, 0, 2)).sum())
        L = lam.detach().double()
        e1, e2 = (L[0] * L[1]).sum().exp(), (L[2] * L[3]).sum().exp()
        unit = torch.stack([e1 * L[1], e1 * L[0], -e2 * L[3], -e2 * L[2]])     # dlam is dw times this
        errors.append(float((dlam * unit).sum() / (unit * unit).sum()) - dw)
    # A row's own f32 roundings (16 terms to a sum of size 0.7, its denominator) are off by 1e-7 or so to either side: 1e-7
    # sqrt(rows) = 2.7e-5 for one seed, half of that for the mean of four; the lean's 7.4e-5 stays in the mean.
    assert abs(sum(errors) / len(errors)) <= 0.5e-9 * rows, errors


@gpu
@pytest.mark.parametrize("shared", [False, True])
def test_lam_at_any_address(shared):
    """A parameter that is a view into a flat buffer starts at any element."""
    q, k, v, lam, do, _ = _inputs(2, 9, 33, 4, 2, 24, F, shared=shared)
    def grads(x):                                                              # noqa: E306
        out = vit_amd.diff_attention(q.cuda(), k.cuda(), v.cuda(), x)
        return out.detach(), torch.autograd.grad(out, x, do.cuda())[0]
    want = grads(lam.cuda().requires_grad_(True))
    for at in (1, 2, 3):
        flat = torch.zeros(lam.numel() + 4, device="cuda")
        flat[at:at + lam.numel()] = lam.cuda().flatten()
        x = flat[at:at + lam.numel()].view(lam.shape).requires_grad_(True)
        assert x.data_ptr() % 16
        assert all(torch.equal(a, b) for a, b in zip(grads(x), want))
        with torch.no_grad():
            out = vit_amd.diff_attention(q.cuda(), k.cuda(), v.cuda(), x)
            assert torch.equal(out, vit_amd.diff_attention(q.cuda(), k.cuda(), v.cuda(), lam.cuda()))


@gpu
def test_broadcast_inputs():
    """Keys that all samples share by a stride of 0: their gradient is the sum over the samples, each rounded to the type."""
    q, k, v, lam, do, _ = _inputs(3, 20, 33, 2, 2, 32, F)
    q, lam, do = q.cuda(), lam.cuda(), do.cuda()
    k1, v1 = k[:1].cuda().requires_grad_(True), v[:1].cuda().requires_grad_(True)
    out = vit_amd.diff_attention(q, k1.expand(3, -1, -1, -1, -1), v1.expand(3, -1, -1, -1), lam)
    dk, dv = torch.autograd.grad(out, (k1, v1), do)
    kf, vf = (t.detach().repeat(3, *[1] * (t.dim() - 1)).requires_grad_(True) for t in (k1, v1))
    full = vit_amd.diff_attention(q, kf, vf, lam)
    assert torch.equal(out, full)
    for a, b in zip((dk, dv), torch.autograd.grad(full, (kf, vf), do)):
        s = b.double().sum(0, keepdim=True)
        assert ((a.double() - s).abs() <= 3 * 2.0 ** -24 * b.double().abs().sum(0, keepdim=True)).all()


@gpu
def test_offsets_past_32_bits():
    """A sample that lies more than 2^32 bytes (and 2^31 elements) behind the first one."""
    far = (1 << 31) + 1024
    d, N, H = 32, 40, 2
    q, k, v, lam, do, _ = (None if t is None else t.cuda() for t in _inputs(2, N, N, H, H, d, H16))
    store = torch.empty(far + N * H * 2 * d, dtype=H16, device="cuda")
    kk = store.as_strided((2, N, H, 2, d), (far, H * 2 * d, 2 * d, d, 1))
    kk.copy_(k)
    a, b = k.requires_grad_(True), kk.requires_grad_(True)
    x, y = vit_amd.diff_attention(q, a, v, lam), vit_amd.diff_attention(q, b, v, lam)
    assert torch.equal(x, y)
    assert torch.equal(torch.autograd.grad(x, a, do)[0], torch.autograd.grad(y, b, do)[0])


@gpu
def test_sizes_with_nothing_to_attend_to():
    lam = torch.randn(4, 16, device="cuda", requires_grad=True)
    for B, nq, nk in ((0, 4, 4), (2, 0, 4), (2, 4, 0)):
        q = torch.randn(B, nq, 2, 2, 16, device="cuda", requires_grad=True)
        k = torch.randn(B, nk, 2, 2, 16, device="cuda", requires_grad=True)
        v = torch.randn(B, nk, 2, 32, device="cuda", requires_grad=True)
        out = vit_amd.diff_attention(q, k, v, lam)
        assert out.shape == (B, nq, 2, 32) and (out == 0).all()
        for g in torch.autograd.grad(out.sum(), (q, k, v, lam)):
            assert (g == 0).all()


@gpu
@pytest.mark.parametrize("case", [(3, 1, 3000, 8, 2, 64), (16, 200, 200, 4, 4, 48), (1, 600, 600, 2, 1, 48)])
def test_streams_capture_and_repeats(case):
    q, k, v, lam, do, _ = (None if t is None else t.cuda() for t in _inputs(*case, H16))
    lens = torch.full((case[0],), case[2], dtype=torch.int32, device="cuda")
    ins = [t.requires_grad_(True) for t in (q, k, v, lam)]

    def step():
        out = vit_amd.diff_attention(*ins, key_lens=lens)
        return [out.detach()] + list(torch.autograd.grad(out, ins, do))
    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b, c in zip(first, other, step()):
        assert torch.equal(a, b) and torch.equal(a, c)
    graphs = []
    for _ in range(2):                                                         # two graphs, replayed at the same time
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        graphs.append((graph, held))
    for i in range(3):
        with torch.no_grad():
            q.copy_(torch.randn(q.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(i)))
            lens.fill_(case[2] - 17 * i)
        side.wait_stream(torch.cuda.current_stream())
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
        torch.cuda.synchronize()
        for a, b, c in zip(graphs[0][1], graphs[1][1], step()):
            assert torch.equal(a, c) and torch.equal(b, c)


@gpu
def test_second_derivatives_are_refused():
    q, k, v, lam, _, _ = (None if t is None else t.cuda() for t in _inputs(1, 3, 4, 1, 1, 8, F))
    q.requires_grad_(True)
    g, = torch.autograd.grad(vit_amd.diff_attention(q, k, v, lam).square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), q)


@gpu
def test_in_place_change_between_the_passes_is_noticed():
    q, k, v, lam, _, _ = (None if t is None else t.cuda() for t in _inputs(1, 3, 4, 1, 1, 8, F))
    q.requires_grad_(True)
    out = vit_amd.diff_attention(q, k, v, lam)
    k.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


# ---- one training step with all of them ------------------------------------------------------------

@gpu
def test_stem_attention_and_clipping_in_one_step():
    """A convolutional stem normalised by group_norm, its map as tokens through the fused projection into diff_attention, a
    loss, the backward pass and clip_grad_norm_: gradients against the same graph of plain f64 operations."""
    torch.manual_seed(0)
    B, S, D, H = 2, 12, 128, 2
    d = D // H // 2
    conv = torch.nn.Conv2d(3, D, 3, padding=1).cuda().to(memory_format=torch.channels_last)
    p = {"gn_w": torch.rand(D) + 0.5, "gn_b": torch.randn(D) * 0.1, "w_in": torch.randn(3 * D, D) * D ** -0.5,
         "lam": torch.randn(4, H, d) * 0.2, "w_out": torch.randn(10, D) * D ** -0.5}
    p = {n: t.cuda().requires_grad_(True) for n, t in p.items()}
    x = torch.randn(B, 3, S, S, device="cuda").to(memory_format=torch.channels_last)
    target = torch.randint(0, 10, (B,), device="cuda")
    params = list(conv.parameters()) + list(p.values())

    def tail(y, mm):                                                          # y: [B, S, S, D], activated
        qkv = mm(y.reshape(B, S * S, D), p["w_in"].to(y.dtype)).view(B, S * S, 3, H, 2 * d)
        return [t for t in qkv.unbind(2)]
    y = vit_amd.group_norm(conv(x).permute(0, 2, 3, 1), 8, p["gn_w"], p["gn_b"], 1e-5, "silu")
    q, k, v = tail(y, lambda a, w: a @ w.t())
    o = vit_amd.diff_attention(q.unflatten(-1, (2, d)), k.unflatten(-1, (2, d)), v, p["lam"], 0.5)
    logits = o.reshape(B, S * S, D).mean(1) @ p["w_out"].t()
    torch.nn.functional.cross_entropy(logits, target).backward()
    got = [t.grad.clone() for t in params]

    ref = [t.detach().double().requires_grad_(True) for t in params]
    cw, cb, gw, gb, wi, lam, wo = ref
    z = torch.nn.functional.conv2d(x.double(), cw, cb, padding=1)
    z = torch.nn.functional.silu(torch.nn.functional.group_norm(z, 8, gw, gb)).permute(0, 2, 3, 1).reshape(B, S * S, D)
    Q, K, V = (z @ wi.t()).view(B, S * S, 3, H, 2 * d).permute(2, 0, 3, 1, 4)
    maps = [(Q[..., m * d:(m + 1) * d] @ K[..., m * d:(m + 1) * d].transpose(-1, -2) * d ** -0.5).softmax(-1) for m in (0, 1)]
    w = ((lam[0] * lam[1]).sum(-1).exp() - (lam[2] * lam[3]).sum(-1).exp() + 0.5).view(1, H, 1, 1)
    o = ((maps[0] - w * maps[1]) @ V).permute(0, 2, 1, 3).reshape(B, S * S, D)
    loss = torch.nn.functional.cross_entropy(o.mean(1) @ wo.t(), target)
    want = torch.autograd.grad(loss, ref)
    for a, b in zip(got, want):
        # f32 products of at most 1,152 terms throughout; the library's convolution and products among them
        assert (a.double() - b).norm() <= 2e-4 * b.norm()
    total = math.sqrt(sum(float(g.double().square().sum()) for g in got))
    norm = vit_amd.clip_grad_norm_(params, 0.1 * total)
    assert abs(float(norm) - total) <= 1e-6 * total
    for t, g in zip(params, got):
        assert (t.grad - 0.1 * g).abs().max() <= 1e-6 * g.abs().max() + 1e-12


# ---- refusals --------------------------------------------------------------------------------------

@gpu
def test_forward_mode_is_refused():
    """A tangent would come back as none at all, which reads as a derivative of zero."""
    from torch.autograd import forward_ad
    tensors = [t.cuda() for t in _inputs(1, 5, 7, 2, 2, 16, F)[:4]]
    with forward_ad.dual_level():
        for i in range(4):
            args = list(tensors)
            args[i] = forward_ad.make_dual(args[i], args[i])
            with pytest.raises(VitkError, match="forward-mode"):
                vit_amd.diff_attention(*args)
        assert vit_amd.diff_attention(*tensors).isfinite().all()


def test_refusals_without_a_gpu():
    t = _inputs(1, 3, 4, 1, 1, 8, F)
    with pytest.raises(VitkError, match="no CPU fallback"):
        vit_amd.diff_attention(*t[:4])
    L = lib.load()
    import ctypes
    p = 1 << 20                                       # never dereferenced: every call below is refused first
    st = (ctypes.c_int64 * 11)(*[64] * 11)
    ok = dict(q=p, out=p, out2=None, lse=None, weight=None, ws=p, floats=1 << 30, batch=2, nq=5, nk=7, heads=4, kv=2, d=32, dtype=0,
              strides=st, lam=p, lam_heads=1, scale=0.1)

    def call(**kw):
        s = {**ok, **kw}
        return L.vitk_diff_attention(s["q"], p, p, s["strides"], s["lam"], s["lam_heads"], 0.5, s["scale"], None, 0, s["out"],
                                     s["out2"], s["lse"], s["weight"], s["ws"], s["floats"], s["batch"], s["nq"], s["nk"],
                                     s["heads"], s["kv"], s["d"], s["dtype"], None)
    assert call(q=None) == 1 and call(out=None) == 1 and call(lam=None) == 1 and call(strides=None) == 1
    assert call(kv=3) == 1 and b"evenly" in L.vitk_last_error()
    assert call(batch=0) == 1 and call(nk=0) == 1 and call(nq=-1) == 1
    assert call(lam_heads=2) == 1
    assert call(dtype=2) == 2
    for d in (0, 4, 12, 72, 128):
        assert call(d=d) == 2
    for s in (0.0, -1.0, float("nan"), float("inf")):
        assert call(scale=s) == 1
    assert call(q=p + 4) == 1 and call(out=p + 8) == 1
    assert call(strides=(ctypes.c_int64 * 11)(*[64] * 10 + [63])) == 1
    assert call(strides=(ctypes.c_int64 * 11)(*[-64] + [64] * 10)) == 1
    assert call(out2=p) == 1
    assert call(batch=1, nk=4096, floats=10) == 1 and b"needed" in L.vitk_last_error()
    assert call(nq=1 << 29) == 2
    assert L.vitk_diff_attention_workspace(2, 5, 7, 4, 3, 32, 0, 0) == -1
    assert L.vitk_diff_attention_workspace(2, 5, 7, 4, 2, 36, 0, 1) == -1

    def back(**kw):
        s = {**ok, **kw}
        return L.vitk_diff_attention_backward(p, p, p, st, p, 1, 0.1, None, 0, p, s.get("o2", p), p, p, p, s.get("dq", p), p, p,
                                              s.get("gs", st), None, s["ws"], s["floats"], 2, 5, 7, 4, 2, 32, 0, None)
    assert back(o2=None) == 1 and back(ws=None) == 1 and back(floats=3) == 1
    assert back(dq=p + 4) == 1
    assert back(gs=(ctypes.c_int64 * 11)(*[2] * 11)) == 1


@gpu
def test_refusals():
    q, k, v, lam, _, _ = (None if t is None else t.cuda() for t in _inputs(2, 5, 7, 4, 2, 16, F))
    ok = dict(q=q, k=k, v=v, lam=lam)
    lens = torch.tensor([1, 2], dtype=torch.int32, device="cuda")
    for bad in (dict(q=q.half(), k=k.half(), v=v.half()), dict(q=q.to(H16)), dict(q=q[..., :1, :]), dict(k=k[:1]), dict(v=v[..., :16]),
                dict(k=k[:, :, [0, 0, 0]], v=v[:, :, [0, 0, 0]]), dict(lam=lam[:3]), dict(lam=lam.to(H16)), dict(lam=lam[:, :2]),
                dict(lam=lam.cpu()), dict(v=v.cpu()), dict(key_lens=lens.long()), dict(key_lens=lens[:1]), dict(key_lens=lens.cpu()),
                dict(scale=0.0), dict(scale=-1.0), dict(q=q.transpose(3, 4).contiguous().transpose(3, 4)),
                dict(q=torch.randn(2, 5, 4, 2, 19, device="cuda")[..., :16]),
                dict(q=q[..., :12], k=k[..., :12], v=v[..., :24], lam=lam[..., :12].contiguous())):
        with pytest.raises(VitkError):
            vit_amd.diff_attention(**{**ok, **bad})


@gpu
def test_sizes_beyond_the_counters_are_refused():
    q = torch.zeros(1, 1, 1, 2, 8, device="cuda", dtype=H16)
    k = q.expand(1, 2 ** 32 + 8, 1, 2, 8)
    v = torch.zeros(1, 1, 1, 16, device="cuda", dtype=H16).expand(1, 2 ** 32 + 8, 1, 16)
    with pytest.raises(VitkError, match="too large"):
        vit_amd.diff_attention(q, k, v, torch.zeros(4, 8, device="cuda"))
    with pytest.raises(VitkError):                                             # fits the counter, not the kernels
        vit_amd.diff_attention(q, k[:, :2 ** 28 + 1], v[:, :2 ** 28 + 1], torch.zeros(4, 8, device="cuda"))
