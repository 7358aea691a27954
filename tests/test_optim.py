"""optim.orthogonalize and optim.Muon against the formulas in float64.

Tolerance of a step: operands in 22 bits with the product of the low parts dropped (2^-21 a product), float32 sums.  An error
made in one step is carried by the derivative of the polynomial, at most a = 3.4445 per step where singular values are small
and below 4 elsewhere, so five steps carry the first one's by at most 4^5; all of them together by 4^5 * 4/3.  Each step's
own error, in the Frobenius norm of X, is at most 8 * 2^-21 sqrt(terms) (three products, coefficients of size 5): the bound is
4^5 * 4/3 * 8 * 2^-21 = 5.2e-3 of the input's norm, which is 1 after the division -- against results whose norm is sqrt(rank).
Measured errors are far smaller because small singular directions are lost relative to themselves, not to the norm; what the
tests allow is 2e-5 of the result's norm per singular-value decade of spread plus half a step of the type."""
import math
import os

import pytest
import torch

from conftest import ROOT  # noqa: F401

DEV = "cuda:0"
CO = (3.4445, -4.7750, 2.0315)
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _oracle(g, steps=5, co=CO, eps=1e-7):
    x = g.double().cpu()
    x = x / (x.square().sum(dim=(-2, -1), keepdim=True).sqrt() + eps)
    for _ in range(steps):
        if x.shape[-2] <= x.shape[-1]:
            a = x @ x.mT
            x = co[0] * x + (co[1] * a + co[2] * (a @ a)) @ x
        else:
            a = x.mT @ x
            x = co[0] * x + x @ (co[1] * a + co[2] * (a @ a))
    return x


def _error(got, want):
    return float((got.double().cpu() - want).norm() / max(float(want.norm()), 1e-300))


def _update(shape, dtype, seed, kind="gauss"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g)
    if kind == "decay":                      # a spectrum of three decades
        u, s, v = torch.linalg.svd(x.double(), full_matrices=False)
        k = s.shape[-1]
        x = ((u * torch.logspace(0, -3, k, dtype=torch.float64)) @ v).float()
    elif kind == "few":                      # a few strong directions over noise
        m, n = shape[-2:]
        x = 0.01 * x + torch.randn(*shape[:-2], m, 3, generator=g) @ torch.randn(*shape[:-2], 3, n, generator=g)
    return x.to(dtype).to(DEV)


SHAPES = [(1, 1), (1, 7), (7, 1), (2, 2), (5, 3), (3, 5), (16, 16), (64, 147), (65, 64), (64, 64), (63, 130), (128, 128),
          (129, 257), (257, 129), (200, 1000), (1000, 200), (2, 33, 17), (3, 1, 40, 72), (384, 384), (64, 576), (576, 64), (20, 3001),
          (100, 129),
          (128, 1152), (2, 1153, 127), (3, 33, 1200), (60, 4111), (4111, 60), (65, 300), (96, 100), (40, 128, 97), (33, 120, 128),
          (64, 320), (449, 31), (7, 30, 640), (40, 16, 500)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_against_float64(shape, dtype):
    from depth_estimation_amd import optim
    for kind in ("gauss", "decay", "few"):
        g = _update(shape, dtype, seed=sum(shape), kind=kind)
        out = optim.orthogonalize(g)
        assert out.shape == g.shape and out.dtype == dtype
        assert _error(out, _oracle(g)) <= 2e-5 * (4 if kind == "decay" else 2) + U[dtype], kind


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(700, 700), (1100, 300), (300, 2049)], ids=str)
def test_larger_tiles(shape):
    from depth_estimation_amd import optim
    g = _update((20,) + shape if shape[0] < 600 else shape, torch.float32, seed=1)
    assert _error(optim.orthogonalize(g), _oracle(g)) <= 4e-5


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["gauss", "decay", "few"])
@pytest.mark.parametrize("shape", [(256, 256), (256, 1000), (1001, 259), (2, 300, 530), (512, 512), (2, 513, 1031), (700, 700),
                                   (1500, 650), (2300, 2100)], ids=str)
def test_bfloat16_with_fewer_products(shape, kind):
    """Sides of 512 and more: 11-bit operands (22 below).  Rounding the result alone is off by 2^-8 / sqrt(3) at most in norm (1.7e-3 for
    numbers spread evenly between powers of two), the operands' rounding by less (9e-4 was the most over these spectra when
    the arithmetic was written out in float64): together at most sqrt(1.7^2 + 1.1^2) 1e-3 = 2.0e-3 with some room, against
    half a step of bfloat16, 3.9e-3."""
    from depth_estimation_amd import optim
    if shape[-1] > 2000 and kind == "decay":
        pytest.skip("a float64 decomposition of this size takes too long")
    g = _update(shape, torch.bfloat16, seed=sum(shape), kind=kind)
    assert _error(optim.orthogonalize(g), _oracle(g)) <= 2.3e-3


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [0, 1, 2, 7])
def test_steps_coefficients_and_eps(steps):
    from depth_estimation_amd import optim
    for shape in ((20, 50), (50, 20)):
        g = _update(shape, torch.float32, seed=steps)
        for co, eps in ((CO, 1e-7), ((1.875, -1.25, 0.375), 0.5), ((1.5, -0.5, 0.0), 0.0)):
            assert _error(optim.orthogonalize(g, steps=steps, coefficients=co, eps=eps), _oracle(g, steps, co, eps)) <= 8e-5


@pytest.mark.gpu
def test_singular_values_end_near_one():
    from depth_estimation_amd import optim
    s = torch.linalg.svdvals(optim.orthogonalize(_update((100, 300), torch.float32, 3)).cpu().double())
    assert 0.6 < float(s.min()) and float(s.max()) < 1.3


@pytest.mark.gpu
def test_zeros_scales_layouts_and_non_finite():
    from depth_estimation_amd import optim
    z = torch.zeros(30, 40, device=DEV)
    assert not optim.orthogonalize(z).any()
    g = _update((48, 80), torch.float32, 4)
    base = optim.orthogonalize(g, eps=0.0)
    for f in (2.0 ** 60, 2.0 ** -60, 2.0 ** -100):      # the norm is taken in float64: no size is lost
        assert torch.equal(optim.orthogonalize(g * f, eps=0.0), base)
    wide = torch.zeros(48, 99, device=DEV)
    wide[:, 3:83] = g
    assert torch.equal(optim.orthogonalize(wide[:, 3:83], eps=0.0), base)
    assert torch.equal(optim.orthogonalize(g.t().contiguous().t(), eps=0.0), base)
    shifted = torch.zeros(48 * 80 + 1, device=DEV)
    shifted[1:] = g.reshape(-1)
    assert torch.equal(optim.orthogonalize(shifted[1:].view(48, 80), eps=0.0), base)
    both = torch.stack([g, 3 * z[0].new_ones(48, 80)])
    assert torch.equal(optim.orthogonalize(both, eps=0.0)[0], base)      # a batch's matrices do not see each other
    g[5, 5] = float("nan")
    both = torch.stack([g, wide[:, 3:83]])
    out = optim.orthogonalize(both, eps=0.0)
    assert torch.isnan(out[0]).all() and torch.equal(out[1], base)
    assert optim.orthogonalize(torch.zeros(0, 4, 5, device=DEV)).shape == (0, 4, 5)
    assert optim.orthogonalize(torch.zeros(3, 0, device=DEV)).shape == (3, 0)


@pytest.mark.gpu
def test_streams_and_captured_graphs():
    from depth_estimation_amd import optim
    a, b = _update((64, 147), torch.float32, 5), _update((300, 100), torch.bfloat16, 6)
    want = optim.orthogonalize(a), optim.orthogonalize(b)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graphs = []
    for x in (a, b):
        with torch.cuda.stream(s):
            optim.orthogonalize(x)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = optim.orthogonalize(x)
        graphs.append((g, out))
    for _ in range(3):
        for g, out in graphs:
            out.zero_()
        torch.cuda.synchronize()
        for g, _ in graphs:
            g.replay()
        eager = optim.orthogonalize(a), optim.orthogonalize(b)
        torch.cuda.synchronize()
        for (g, out), w, e in zip(graphs, want, eager):
            assert torch.equal(out, w) and torch.equal(e, w)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("shape", [(1000, 40003), (20003, 1500), (1500, 20003), (300, 65531), (500, 65531), (64, 65531)], ids=str)
def test_long_sides(shape, dtype):
    """Sums over a long side split over many workgroups, with a last split that is short or empty.  The tolerances of
    test_against_float64 and test_bfloat16_with_fewer_products."""
    from depth_estimation_amd import optim
    g = torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(sum(shape)), device=DEV).to(dtype)
    x = g.double()
    x /= x.norm() + 1e-7
    for _ in range(5):
        a = x @ x.mT if shape[0] <= shape[1] else x.mT @ x
        b = CO[1] * a + CO[2] * (a @ a)
        x = CO[0] * x + (b @ x if shape[0] <= shape[1] else x @ b)
    out = optim.orthogonalize(g).double()
    assert float((out - x).norm() / x.norm()) <= (4e-5 if dtype == torch.float32 else 2.3e-3 if min(shape) >= 256 else 4e-5 + U[dtype])


@pytest.mark.gpu
def test_captured_graphs_of_every_form():
    """One workgroup's memory above its default, slabs, split sums: replayed with eager calls between."""
    from depth_estimation_amd import optim
    s = torch.cuda.Stream()
    for shape, dtype in (((128, 128), torch.float32), ((64, 1500), torch.bfloat16), ((2, 300, 700), torch.float32),
                         ((700, 700), torch.bfloat16)):
        x, y = _update(shape, dtype, 7), _update(shape, dtype, 8)
        buf = x.clone()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            optim.orthogonalize(buf)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = optim.orthogonalize(buf)
        for src in (x, y, x):
            buf.copy_(src)
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, optim.orthogonalize(src))


@pytest.mark.gpu
def test_muon_steps():
    """Three steps of a small set of parameters (two of one shape, a convolution, one without a gradient) against the formula."""
    from depth_estimation_amd import optim
    gen = torch.Generator().manual_seed(7)
    shapes = [(30, 20), (30, 20), (16, 3, 7, 7), (8, 8)]
    ps = [torch.nn.Parameter(torch.randn(*s, generator=gen).to(DEV)) for s in shapes]
    lr, mom, wd = 0.05, 0.9, 0.1
    opt = optim.Muon(ps, lr=lr, momentum=mom, weight_decay=wd)
    ref = [p.detach().double().cpu() for p in ps]
    bufs = [torch.zeros_like(r) for r in ref]
    for _ in range(3):
        for i, p in enumerate(ps):
            p.grad = None if i == 3 else torch.randn(p.shape, generator=gen).to(DEV)
        opt.step()
        for i, p in enumerate(ps[:3]):
            g = p.grad.double().cpu()
            bufs[i] = mom * bufs[i] + g
            u = (g + mom * bufs[i]).flatten(1)
            o = _oracle(u.float()).view(p.shape)
            ref[i] = ref[i] * (1 - lr * wd) - lr * max(1.0, u.shape[0] / u.shape[1]) ** 0.5 * o
    for i, p in enumerate(ps):
        assert _error(p.detach(), ref[i]) <= 1e-4
    state = opt.state_dict()
    other = optim.Muon(ps, lr=lr)
    other.load_state_dict(state)
    assert torch.equal(other.state[ps[0]]["momentum_buffer"], opt.state[ps[0]]["momentum_buffer"])


@pytest.mark.gpu
def test_whole_training_step_with_matrix_updates():
    """scripts/full_step.train_step with --optimizer muon: every matrix moves by its orthogonalised first momentum, the vectors
    by Adam."""
    import depth_estimation_amd as de
    from scripts import full_step as fs
    dev, H, W = torch.device(DEV), 48, 160
    nets = fs.build_networks(dev, dict(pose=20_000, decoder=1_000, convgru=500), seed=3)
    params = fs.trainable(nets)
    before = [p.detach().clone() for p in params]
    opt = fs.build_optimizer(params, "muon")
    imgs = torch.rand(1, 3, 3, H, W, generator=torch.Generator().manual_seed(9)).to(dev)
    loss = fs.train_step(nets, opt, None, imgs, fs.hip_path(de, H, W, dev))
    assert bool(torch.isfinite(loss))
    for p, old in zip(params, before):
        if p.dim() < 2:
            assert float((p - old).abs().max()) <= 1.01e-3                      # Adam's first step: at most its learning rate
            continue
        g = p.grad.flatten(1)
        want = _oracle(1.95 * g).view(p.shape).to(dev) * 0.02 * max(1.0, g.shape[0] / g.shape[1]) ** 0.5
        # the orthogonalised matrix is exact to 2e-4 of its norm (the gradients' spectra are wide); a step of size 0.02 on
        # weights of size one is read back with 2^-24
        assert float(((old - p.detach()).double() - want).norm()) <= 1e-3 * float(want.norm()) + 2.0 ** -24 * p.numel() ** 0.5


def test_refusals_on_the_host():
    from depth_estimation_amd import _lib as L, optim
    with pytest.raises(RuntimeError, match="GPU"):
        optim.orthogonalize(torch.zeros(4, 4))
    with pytest.raises(ValueError):
        optim.Muon([torch.nn.Parameter(torch.zeros(4))])
    muon = optim.Muon([torch.nn.Parameter(torch.zeros(4, 4))])
    with pytest.raises(ValueError):
        muon.add_param_group(dict(params=[torch.nn.Parameter(torch.zeros(4))]))
    assert len(muon.param_groups) == 1
    for bad in (dict(lr=-1.0), dict(momentum=1.0), dict(weight_decay=-0.1)):
        with pytest.raises(ValueError):
            optim.Muon([torch.nn.Parameter(torch.zeros(4, 4))], **bad)
    if not os.path.exists(L.LIB_PATH):
        pytest.skip("libdepthsynth.so not built (run __graft_entry__.build())")
    import ctypes as C
    lib, fake, co = L.lib(), 0x1000, (C.c_double * 3)(*CO)

    def call(u=fake, dt=0, b=1, m=8, n=8, steps=5, c=co, eps=1e-7, out=fake, ws=fake, nb=1 << 40):
        return lib.ds_orthogonalize(u, dt, b, m, n, steps, c, eps, out, ws, nb, None)

    for rc, want in [(call(u=None), -1), (call(out=None), -1), (call(c=None), -1), (call(steps=-1), -1), (call(eps=-1.0), -1),
                     (call(eps=math.nan), -1), (call(b=0), -1), (call(m=0), -1), (call(n=-3), -1), (call(dt=3), -2),
                     (call(steps=33), -2), (call(m=1 << 17), -2), (call(m=40000, n=40000), -2), (call(b=70000), -2),
                     (call(ws=None), -3), (call(nb=16), -3), (call(ws=fake + 8), -3), (call(out=fake + 4), -1)]:
        assert rc == want
    assert lib.ds_orthogonalize_workspace_bytes(0, 1, 0, 4) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["gauss", "decay", "few"])
@pytest.mark.parametrize("co,steps", [(CO, 1), (CO, 6), (CO, 7), (CO, 10), (CO, 32), ((3.3, -5.79, 2.49), 6), ((3.37, -4.33, 1.38), 6),
                                      ((4.08, -6.89, 2.93), 5), ((1.875, -1.25, 0.375), 12), ((2.09, -2.52, 1.28), 6)], ids=str)
def test_bfloat16_of_any_steps_and_coefficients(co, steps, kind):
    """The tolerance of test_bfloat16_with_fewer_products whatever the steps and the polynomial: 1.7e-3 for the result's rounding
    and 1.2e-3 for 11-bit operands where they are taken make 2.1e-3.  Where 22 bits are kept, their 2^-21 a product, carried
    through steps that multiply it by less than 4 while small singular values grow and by 1.6 near the polynomial's fixed
    points, stays below 1e-4."""
    from depth_estimation_amd import optim
    g = _update((520, 600), torch.bfloat16, seed=steps, kind=kind)
    assert _error(optim.orthogonalize(g, steps=steps, coefficients=co), _oracle(g, steps, co)) <= 2.3e-3


# coefficients, steps: singular values grow to 3 and fall to 0; wander up to 3.2; double, quadruple; grow a thousandfold, and
# by 4 and more (2^20 and beyond); shrink a thousandfold
REACHES = [((3.375, -0.375, 0.0), 2), ((2.6, -0.25, 0.0), 5), ((2.0, 0.0, 0.0), 5), ((4.0, 0.0, 0.0), 3), ((10.0, 0.0, 0.0), 4),
           ((1.0, 2.0, 0.5), 3), ((-3.0, -1.0, 0.0), 3), ((0.1, 0.0, 0.0), 4), ((0.0, 0.0, 1.5), 3), ((0.0, 0.0, 0.0), 2)]


@pytest.mark.gpu
@pytest.mark.parametrize("co,steps", REACHES, ids=str)
@pytest.mark.parametrize("shape", [(1, 1), (3, 5), (40, 60), (40, 700), (130, 90), (3, 200, 300)], ids=str)
def test_coefficients_that_take_singular_values_far(co, steps, shape):
    """In the Frobenius norm.  A step takes values of at most m to at most M = |a| m + |b| m^3 + |c| m^5 and errors to at most
    L = |a| + 3 |b| m^2 + 5 |c| m^4 times themselves.  Its own error: three products of 22-bit operands (2^-21 each) with float32
    sums, of matrices of norm m sqrt(k) at most whose absolute values' norms are sqrt(k) times theirs at most: 6 2^-21 k M."""
    from depth_estimation_amd import optim
    k = min(shape[-2:])
    one_entry = torch.zeros(shape, device=DEV)
    one_entry[..., 0, 0] = 1.0                       # rank one, along an axis: one entry holds the whole singular value
    for g in (_update(shape, torch.float32, seed=3), one_entry, -one_entry):
        want = _oracle(g, steps, co)
        m, tol = 1.0, 0.0
        for _ in range(steps):
            a, b, c = (abs(x) for x in co)
            big = a * m + b * m ** 3 + c * m ** 5
            tol = tol * (a + 3 * b * m ** 2 + 5 * c * m ** 4) + 6 * 2.0 ** -21 * k * big
            m = big
        got = optim.orthogonalize(g, steps=steps, coefficients=co)
        assert bool(torch.isfinite(got).all())
        assert float((got.double().cpu() - want).norm()) <= tol * math.prod(shape[:-2]) ** 0.5 + 2.0 ** -24 * float(want.norm())


@pytest.mark.gpu
def test_coefficients_at_their_limit():
    from depth_estimation_amd import optim
    one = torch.ones(1, 1, device=DEV)
    for co, steps in (((2.0 ** 24, 0.0, 0.0), 2), ((2.0, 0.0, 0.0), 25)):        # 2^24 before the last step
        got = optim.orthogonalize(one, steps=steps, coefficients=co, eps=0.0)
        assert abs(float(got) / co[0] ** steps - 1) <= steps * 2.0 ** -21
    for co, steps in (((2.0 ** 24, 0.0, 0.0), 3), ((2.0, 0.0, 0.0), 26), ((2.0 ** 24 + 4, 0.0, 0.0), 2), ((0.0, 0.0, 10.0 ** 31), 1)):
        with pytest.raises(RuntimeError):
            optim.orthogonalize(one, steps=steps, coefficients=co, eps=0.0)


def test_refusals_of_coefficients_on_the_host():
    from depth_estimation_amd import _lib as L
    if not os.path.exists(L.LIB_PATH):
        pytest.skip("libdepthsynth.so not built (run __graft_entry__.build())")
    import ctypes as C
    lib, fake = L.lib(), 0x1000
    for co, steps, want in (((3.0, 0.0, 0.0), 32, -2), ((2.0 ** 30, 0.0, 0.0), 2, -2), ((0.0, 0.0, 1e200), 1, -2),
                            ((math.nan, 0.0, 0.0), 1, -1), ((1.0, math.inf, 0.0), 1, -1)):
        assert lib.ds_orthogonalize(fake, 0, 1, 8, 8, steps, (C.c_double * 3)(*co), 0.0, fake, fake, 1 << 40, None) == want


def test_muon_refuses_on_the_host():
    from depth_estimation_amd import optim
    ok = torch.nn.Parameter(torch.zeros(4, 4))
    meta = torch.device("meta")
    for p in (torch.empty(100_000, 8, device=meta), torch.empty(8, 70_000, device=meta), torch.empty(40_000, 40_000, device=meta),
              torch.empty(8, 300, 300, device=meta), torch.empty(4, 4, dtype=torch.float64),
              torch.empty(4, 4, dtype=torch.complex64)):
        p = torch.nn.Parameter(p)
        with pytest.raises(ValueError):
            optim.Muon([ok, p])
        muon = optim.Muon([ok])
        with pytest.raises(ValueError):
            muon.add_param_group(dict(params=[p]))
        assert len(muon.param_groups) == 1
    for bad in (dict(steps=-1), dict(steps=33), dict(coefficients=(1.0, 2.0)), dict(coefficients=(1.0, math.nan, 0.0)),
                dict(eps=-1.0)):
        with pytest.raises(ValueError):
            optim.Muon([ok], **bad)
    optim.Muon([torch.nn.Parameter(torch.empty(65536, 32768, device=meta)), torch.nn.Parameter(torch.empty(0, 5))])


def test_muon_step_that_cannot_be_made_changes_nothing():
    """One gradient of two is on the CPU, sparse, or the options are out of range: no buffer, no parameter moves."""
    from depth_estimation_amd import optim
    for how in ("cpu", "sparse", "steps"):
        ps = [torch.nn.Parameter(torch.ones(4, 4)) for _ in range(2)]
        muon = optim.Muon(ps)
        for p in ps:
            p.grad = torch.ones(4, 4)
        if how == "sparse":
            ps[0].grad = ps[0].grad.to_sparse()
        if how == "steps":
            muon.param_groups[0]["steps"] = 40
        for _ in range(2):
            with pytest.raises(RuntimeError):
                muon.step()
        assert all(torch.equal(p, torch.ones(4, 4)) for p in ps) and not muon.state


@pytest.mark.gpu
def test_muon_second_group_refused_before_the_first_moves():
    from depth_estimation_amd import optim
    a, b = (torch.nn.Parameter(torch.ones(6, 5, device=DEV)) for _ in range(2))
    muon = optim.Muon([dict(params=[a]), dict(params=[b], coefficients=(3.0, 0.0, 0.0), steps=32)])      # beyond 2^24
    a.grad, b.grad = torch.ones_like(a), torch.ones_like(b)
    with pytest.raises(RuntimeError):
        muon.step()
    assert torch.equal(a, torch.ones_like(a)) and not muon.state
    muon.param_groups[1]["steps"] = 5
    muon.step()
    assert not torch.equal(a, torch.ones_like(a)) and torch.equal(muon.state[a]["momentum_buffer"], a.grad)


@pytest.mark.gpu
def test_refusals_of_tensors():
    from depth_estimation_amd import optim
    g = torch.zeros(4, 4, device=DEV)
    for args, kw in [((g[0],), {}), ((g.double(),), {}), ((g.int(),), {}), ((g,), dict(steps=-1)), ((g,), dict(steps=40)), ((g,), dict(steps=2 ** 32 + 5)),
                     ((g,), dict(coefficients=(1.0, 2.0))), ((g,), dict(coefficients=(1.0, 2.0, math.inf))),
                     ((g,), dict(eps=-1.0)), ((g,), dict(eps=math.nan))]:
        with pytest.raises(RuntimeError):
            optim.orthogonalize(*args, **kw)
