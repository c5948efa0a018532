"""Global gradient norm and clipping (vit_amd.grad_norm, vit_amd.clip_grad_norm_) against 64-bit arithmetic."""
import ctypes
import math

import pytest
import torch

import vit_amd
from vit_amd import VitkError, lib

gpu = pytest.mark.gpu
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def _params(sizes, dtypes, seed=0, scale=1e-2, offset=0):
    """Parameters with gradients; offset > 0: views that start at odd elements of one buffer per type, guard values
    between them."""
    gen = torch.Generator().manual_seed(seed)
    out = []
    for s, t in zip(sizes, dtypes):
        g = (torch.randn(s, generator=gen) * scale).to(t).cuda()
        if offset:
            held = torch.full((s + 2 * offset,), 7.0, dtype=t, device="cuda")
            held[offset:offset + s] = g
            g = held[offset:offset + s]
            g._held = held
        p = torch.zeros(s, dtype=t, device="cuda").requires_grad_(True)
        p.grad = g
        out.append(p)
    return out


def _norm64(params):
    return math.sqrt(math.fsum(float(p.grad.double().square().sum()) for p in params))


def _check_clip(params, max_norm, **kw):
    before = [p.grad.double().cpu() for p in params]
    want = math.sqrt(math.fsum(float(g.square().sum()) for g in before))
    ptrs = [p.grad.data_ptr() for p in params]
    norm = vit_amd.clip_grad_norm_(params, max_norm, **kw)
    assert norm.dtype == torch.float32 and norm.shape == ()
    if want < torch.finfo(torch.float32).max:
        assert abs(float(norm) - want) <= 2 ** -23 * want                  # f64 sum, one rounding
    else:
        assert float(norm) == math.inf                                     # what f32 rounds it to; the factor is finite
    c = min(1.0, max_norm / (want + 1e-6))
    for p, g, a in zip(params, before, ptrs):
        assert p.grad.data_ptr() == a
        got, t = p.grad.double().cpu(), p.grad.dtype
        if c == 1.0:
            assert torch.equal(got, g)
        else:
            # the factor's rounding, the product's, the type's; below the normal range the last one is absolute
            assert ((got - g * c).abs() <= (g * c).abs() * (HALF[t] + 2 * 2.0 ** -24) + torch.finfo(t).smallest_normal * HALF[t]).all()
    return norm


F, H = torch.float32, torch.bfloat16
LISTS = {
    "one": ([1], [F]),
    "small": ([1, 2, 3, 5, 7, 8, 9, 15, 17, 31], [F, H] * 5),
    "odd": ([1000, 65537, 16384, 16385, 131072 + 3, 333], [H, F, F, H, H, F]),
    "zero_sized": ([0, 5, 0, 100, 0], [F, F, H, H, F]),
    "over_one_launch": ([(37 * i) % 211 + 1 for i in range(400)], [F, H, F, F] * 100),
    "large": ([3_000_001, 768, 2_000_000, 12], [F, F, H, H]),
}


@gpu
@pytest.mark.parametrize("offset", [0, 1, 3])
@pytest.mark.parametrize("name", LISTS)
def test_clips_to_the_bound(name, offset):
    sizes, dtypes = LISTS[name]
    params = _params(sizes, dtypes, offset=offset)
    want = _norm64(params)
    _check_clip(params, 0.3 * want)
    assert abs(_norm64(params) - 0.3 * want) <= 2 ** -8 * want
    if offset:
        for p in params:
            held = p.grad._held
            assert (held[:offset] == 7).all() and (held[held.numel() - offset:] == 7).all()


@gpu
@pytest.mark.parametrize("name", LISTS)
def test_leaves_gradients_under_the_bound_alone(name):
    params = _params(*LISTS[name], offset=1)
    _check_clip(params, 1.01 * _norm64(params) + 1e-5)


@gpu
def test_norm_alone_and_the_largest_magnitude():
    params = _params([10_000, 3, 77], [F, H, F], seed=4)
    grads = [p.grad for p in params]
    assert abs(float(vit_amd.grad_norm(grads)) - _norm64(params)) <= 2 ** -23 * _norm64(params)
    assert float(vit_amd.grad_norm(grads, math.inf)) == max(float(g.abs().max()) for g in grads)
    assert float(vit_amd.grad_norm(grads[0])) == float(vit_amd.grad_norm([grads[0]]))
    top = float(vit_amd.grad_norm(grads, float("inf")))
    before = [g.double().clone() for g in grads]
    assert float(vit_amd.clip_grad_norm_(params, 0.5 * top, norm_type=math.inf)) == top
    c = 0.5 * top / (top + 1e-6)
    for g, h in zip(grads, before):
        assert ((g.double() - c * h).abs() <= (c * h).abs() * (HALF[g.dtype] + 2 ** -23)).all()


@gpu
@pytest.mark.parametrize("scale", [1e30, 1e-30, 3e37])
def test_magnitudes_whose_squares_leave_f32(scale):
    params = _params([4096, 33], [F, H], scale=scale)
    _check_clip(params, 1.0)


@gpu
def test_zero_and_absent_gradients_and_bounds():
    params = _params([100, 7], [F, H], scale=0.0)
    assert float(vit_amd.clip_grad_norm_(params, 1.0)) == 0.0
    assert all((p.grad == 0).all() for p in params)
    params = _params([100, 7], [F, H])
    for p in params:
        p.grad = None
    assert float(vit_amd.clip_grad_norm_(params, 1.0)) == 0.0
    assert float(vit_amd.clip_grad_norm_([], 1.0)) == 0.0
    empty = torch.zeros(0, device="cuda", requires_grad=True)
    empty.grad = torch.zeros(0, device="cuda")
    assert float(vit_amd.clip_grad_norm_([empty], 1.0)) == 0.0
    one = _params([50], [F])[0]
    vit_amd.clip_grad_norm_(one, 0.0)                                      # a single parameter; a bound of 0
    assert (one.grad == 0).all()


@gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("kind", [2.0, math.inf])
def test_non_finite_gradients_follow_torch(bad, kind):
    for where in (0, 1):
        params, mirror = _params([70_000, 9], [F, H], seed=3), _params([70_000, 9], [F, H], seed=3)
        for q in (params, mirror):
            q[where].grad[5] = bad
        norm = vit_amd.clip_grad_norm_(params, 1.0, norm_type=kind)
        assert math.isnan(float(norm)) if bad != bad else float(norm) == math.inf
        want = torch.nn.utils.clip_grad_norm_(mirror, 1.0, norm_type=kind)
        assert torch.equal(torch.isnan(norm.cpu()), torch.isnan(want.float().cpu()))
        for p, m in zip(params, mirror):
            assert torch.equal(p.grad.isnan(), m.grad.isnan())
            ok = ~p.grad.isnan()
            assert torch.equal(p.grad[ok], m.grad[ok])
    params = _params([70_000, 9], [F, H], seed=3)
    params[1].grad[5] = bad
    before = [p.grad.clone() for p in params]
    with pytest.raises(VitkError, match="cannot be clipped"):
        vit_amd.clip_grad_norm_(params, 1.0, norm_type=kind, error_if_nonfinite=True)
    for p, g in zip(params, before):
        assert torch.equal(p.grad.isnan(), g.isnan()) and torch.equal(p.grad.nan_to_num(), g.nan_to_num())


@gpu
def test_error_if_nonfinite_clips_finite_gradients():
    params = _params([1000, 7], [F, H])
    _check_clip(params, 0.1, error_if_nonfinite=True)


@gpu
def test_permuted_dense_gradients_and_refused_strides():
    p = torch.zeros(8, 6, 5, 7, device="cuda").to(memory_format=torch.channels_last).requires_grad_(True)
    p.grad = torch.randn(8, 6, 5, 7, device="cuda").to(memory_format=torch.channels_last)
    _check_clip([p], 0.5)
    q = torch.zeros(10, 10, device="cuda", requires_grad=True)
    q.grad = torch.randn(10, 20, device="cuda")[:, ::2]
    with pytest.raises(VitkError, match="fill its memory"):
        vit_amd.clip_grad_norm_([q], 1.0)
    q.grad = torch.randn(10, 1, device="cuda").expand(10, 10)
    with pytest.raises(VitkError, match="fill its memory"):
        vit_amd.clip_grad_norm_([q], 1.0)


@gpu
def test_shared_memory_and_types_are_refused():
    a, b = _params([100, 100], [F, F])
    with pytest.raises(VitkError, match="share memory"):
        vit_amd.clip_grad_norm_([a, b, a], 1.0)
    b.grad = a.grad
    with pytest.raises(VitkError, match="share memory"):
        vit_amd.clip_grad_norm_([b, a], 1.0)
    h = torch.zeros(5, device="cuda", dtype=torch.float16, requires_grad=True)
    h.grad = torch.ones_like(h)
    with pytest.raises(VitkError, match="bf16 or f32"):
        vit_amd.clip_grad_norm_([h], 1.0)
    c = torch.zeros(5, requires_grad=True)
    c.grad = torch.ones(5)
    with pytest.raises(VitkError, match="one CUDA/HIP device"):
        vit_amd.clip_grad_norm_([a, c], 1.0)


@gpu
def test_runs_on_another_stream_and_in_a_captured_graph():
    params = _params([100_003, 5, 4096], [F, H, F])
    source = [p.grad.clone() for p in params]
    bound = 0.25 * _norm64(params)
    _check_clip(params, bound)
    want = [p.grad.clone() for p in params]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for p, g in zip(params, source):
            p.grad.copy_(g)
        vit_amd.clip_grad_norm_(params, bound)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p.grad, w) for p, w in zip(params, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = vit_amd.clip_grad_norm_(params, bound)
    for i in range(4):
        f = 1.0 + i                                                        # other gradients, the same addresses
        for p, g in zip(params, source):
            p.grad.copy_(g.float() * f)
        eager = _params([100_003, 5, 4096], [F, H, F])
        for p, q in zip(eager, params):
            p.grad = q.grad.clone()
        wn = vit_amd.clip_grad_norm_(eager, bound)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, wn)
        assert all(torch.equal(p.grad, q.grad) for p, q in zip(params, eager))


@gpu
def test_a_graph_that_saved_a_gradient_notices_the_clipping():
    a, b = _params([64, 7], [F, H])
    saved = torch.ones(64, device="cuda", requires_grad=True)
    for bound in (0.25 * _norm64([a, b]), 4.0 * _norm64([a, b])):              # scaled, and under the bound
        versions = a.grad._version, b.grad._version
        out = (saved * a.grad).sum()
        vit_amd.clip_grad_norm_([a, b], bound)
        assert a.grad._version > versions[0] and b.grad._version > versions[1]
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.backward()
    with torch.inference_mode():                                               # tensors without a counter
        p = torch.zeros(5, device="cuda")
        p.grad = torch.ones(5, device="cuda")
        vit_amd.clip_grad_norm_([p], 1.0)
        assert abs(float(p.grad.norm()) - 1.0) < 1e-5


# ---- refusals that touch no GPU --------------------------------------------------------------------

def _list(addr, size, kind):
    n = len(addr)
    return (ctypes.c_uint64 * n)(*addr), (ctypes.c_int64 * n)(*size), (ctypes.c_int * n)(*kind), n


def test_refusals_without_a_gpu():
    with pytest.raises(VitkError, match="CUDA/HIP"):
        vit_amd.grad_norm([torch.ones(4)])
    p = torch.zeros(4, requires_grad=True)
    p.grad = torch.ones(4)
    with pytest.raises(VitkError, match="CUDA/HIP"):
        vit_amd.clip_grad_norm_([p], 1.0)
    for bad in (-1.0, float("nan")):
        with pytest.raises(VitkError, match="max_norm"):
            vit_amd.clip_grad_norm_([p], bad)
    with pytest.raises(VitkError, match="norm_type"):
        vit_amd.clip_grad_norm_([p], 1.0, norm_type=3)
    assert float(vit_amd.clip_grad_norm_([], 1.0)) == 0.0 and float(vit_amd.grad_norm([])) == 0.0
    L = lib.load()
    assert L.vitk_grad_norm_workspace(0) == 0 and L.vitk_grad_norm_workspace(-1) == -1
    assert L.vitk_grad_norm_workspace(184) * 2 == L.vitk_grad_norm_workspace(185)
    ws, part = 1 << 20, 4096                               # addresses are compared, never read

    def clip(addr, size, kind, norm_kind=0, max_norm=1.0, n_partials=ws, partials=part):
        return L.vitk_grad_clip(*_list(addr, size, kind), norm_kind, partials, n_partials, max_norm, None, None)
    assert clip([4096, 4096], [4, 4], [0, 0]) == 1 and b"share memory" in L.vitk_last_error()
    assert clip([8192, 4096], [4, 1025], [0, 0]) == 1 and b"share memory" in L.vitk_last_error()
    assert clip([4096, 8192, 4100], [8, 4, 2], [1, 0, 1]) == 1 and b"share memory" in L.vitk_last_error()
    assert clip([4096], [4], [2]) == 2
    assert clip([4098], [4], [0]) == 1 and b"misaligned" in L.vitk_last_error()
    assert clip([0], [4], [0]) == 1
    assert clip([4096], [-4], [0]) == 1
    assert clip([4096], [4], [0], norm_kind=2) == 1
    assert clip([4096], [4], [0], max_norm=-1.0) == 1
    assert clip([4096], [4], [0], max_norm=float("nan")) == 1
    assert clip([4096], [4], [0], n_partials=10) == 1
    assert clip([4096], [4], [0], partials=None) == 1
    assert L.vitk_grad_norm(*_list([4096], [4], [0]), 0, None, ws, None, None) == 1
    assert L.vitk_grad_norm(None, None, None, 3, 0, part, ws, None, None) == 1


def test_sizes_beyond_the_piece_counter_are_refused():
    """A tensor of more than 2^31 pieces was never cut: the host went round for good."""
    L = lib.load()
    for size in ([(1 << 46) - 1], [(1 << 42) + 1], [1 << 42, 1], [1 << 41, 1 << 40, 1 << 40, 1]):
        args = _list([4096 << i for i in range(len(size))], size, [lib.VITK_F32] * len(size))
        assert L.vitk_grad_norm(*args, 0, 4096, 1 << 20, None, None) == lib.VITK_ERR_UNSUPPORTED, size
        assert b"16 TiB" in L.vitk_last_error()
        assert L.vitk_grad_clip(*args, 0, 4096, 1 << 20, 1.0, None, None) == lib.VITK_ERR_UNSUPPORTED
