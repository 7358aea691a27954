"""metrics.linear_cross_entropy and synthesis.depth_from_bins against their formulas in float64.

Tolerances, element by element, from the arithmetic (u: half a step of a type, 2^-8 bfloat16, 2^-11 float16, 2^-24 float32):
  * logits: operands exact (16-bit types) or 22 bits with the product of the two low parts dropped (float32: 2^-21 per
    product, plus 2^-40 of the largest operand where a small one's low part runs out of fp16's range); fp32 sums of D terms:
    |dl| <= (2^-21 [float32] + (D + 4) 2^-24) sum_d |h||w| =: e_l;
  * a probability: relative error <= 2 (max_v e_l) (its own logit and the normaliser) + (V + 32) 2^-24 (sum, exponentials whose
    argument carries |l - max| 2^-24 with |l - max| <= 24 where p matters, divisions) =: e_p;
  * dl is rounded to u of the operand type (2^-21 for float32's planes) before the products and summed in fp32:
    |d out| <= sum |dl||x| (u + e_p' + terms 2^-24) + u |out|.
"""
import math
import os

import pytest
import torch

from conftest import ROOT  # noqa: F401

DEV = "cuda:0"
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _data(n, d, v, dtype, seed, keep=1.0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(v, d, generator=g) / math.sqrt(d)
    t = torch.randint(0, v, (n,), generator=g)
    h = spread * torch.randn(n, d, generator=g) + 2.0 * w[t]
    drop = torch.rand(n, generator=g) >= keep
    up = torch.rand(n, generator=g) + 0.5
    c = torch.sort(80 * torch.rand(v, generator=g) + 0.1).values
    return h.to(dtype).to(DEV), w.to(dtype).to(DEV), torch.where(drop, torch.full_like(t, -100), t).to(DEV), up.to(DEV), c.to(DEV)


def _oracle(h, w, t=None, c=None, up=None, ignore=-100):
    """float64: (per-row output, g_hidden, g_weight, and the tolerances of the three) for upstream `up` per row"""
    dt = h.dtype
    n, d = h.shape
    v = w.shape[0]
    H, W, up = h.double(), w.double(), up.double()
    ok = torch.ones(n, dtype=torch.bool, device=h.device) if t is None else t != ignore
    H = torch.where(ok[:, None], H, 0.0)
    l = H @ W.T
    split = 2.0 ** -21 if dt == torch.float32 else 0.0
    # 2^-40 of the largest operand per term, where the low plane underflows
    floor = 2.0 ** -40 * (H.abs().max() if n else 0.0) * W.abs().max() * 2 * d if dt == torch.float32 else 0.0
    el = (split + (d + 4) * 2.0 ** -24) * (H.abs() @ W.abs().T) + floor
    top = el.max(dim=1, keepdim=True).values
    p = torch.softmax(l, dim=1)
    ep = 2 * top + (v + 32) * 2.0 ** -24
    if t is not None:
        tc = t.clamp(min=0)
        one = torch.nn.functional.one_hot(tc, v).double()
        out = torch.where(ok, torch.logsumexp(l, 1) - l.gather(1, tc[:, None])[:, 0], 0.0)
        tol = 2 * top[:, 0] + (v + 32) * 2.0 ** -24 + 4 * 2.0 ** -24 * (l.abs().max(dim=1).values + out.abs() + 1)
        dl = (p - one) * (up * ok)[:, None]
        mag = (p * ep + one * 2.0 ** -24) * (up.abs() * ok)[:, None]      # a bound: the upstream's size, not its sign
    else:
        cd = c.double()
        out = p @ cd
        tol = (ep * (p @ cd.abs())[:, None])[:, 0] + 4 * 2.0 ** -24 * out.abs()
        dl = p * (cd[None] - out[:, None]) * up[:, None]
        mag = p * (ep * (cd[None] - out[:, None]).abs() + tol[:, None] + 2.0 ** -23 * cd.abs()[None]) * up.abs()[:, None]
    ur = 2.0 ** -21 if dt == torch.float32 else U[dt]
    # what dl is stored to: ur of it, or where that is below fp16's normal numbers half a subnormal step, 2^-25.  dl is stored
    # as 2^14 dl / s with s at most twice the largest upstream value (times four times the largest centre): the half step is
    # 2^-25 2^-14 2 = 2^-38 of the largest upstream value -- not of the largest dl, which is smaller where every row is sure
    # of its class
    unit = (up * ok).abs().max() * (1.0 if t is not None else 4 * c.abs().max().double()) if n else 0.0
    err = mag + ur * (dl.abs() + mag) + (0.0 if dt == torch.bfloat16 else 2.0 ** -38 * unit)
    gh, gw = dl @ W, dl.T @ H
    th = (err + (v + 8) * 2.0 ** -24 * dl.abs()) @ W.abs() + U[dt] * gh.abs() + split * (dl.abs() @ W.abs())
    tw = (err + (n + 8) * 2.0 ** -24 * dl.abs()).T @ H.abs() + U[dt] * gw.abs() + split * (dl.abs().T @ H.abs())
    # results below the smallest normal number of the type are rounded to its subnormal steps
    sub = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}[dt]
    return out, gh, gw, tol, th * 1.01 + sub, tw * 1.01 + sub


def _close(got, want, tol, what):
    got = got.double()
    assert got.shape == want.shape, what
    bad = (got - want).abs() - tol
    assert bool((bad <= 0).all()), f"{what}: off by {(got - want).abs().max():.3g}, over its bound by {bad.max():.3g}"


def _ce(h, w, t, reduction="none", up=None, ignore=-100):
    from depth_estimation_amd import metrics
    h, w = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
    out = metrics.linear_cross_entropy(h, w, t, ignore_index=ignore, reduction=reduction)
    gh, gw = torch.autograd.grad(out, (h, w), up)
    return out.detach(), gh, gw


def _ex(h, w, c, up):
    from depth_estimation_amd import synthesis
    h, w = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
    out = synthesis.depth_from_bins(h, w, c)
    gh, gw = torch.autograd.grad(out, (h, w), up)
    return out.detach(), gh, gw


# rows, features, classes: one of each; odd everything; tile edges and one beyond; long reductions on either side; few rows
# against many classes and the reverse
SIZES = [(1, 1, 1), (1, 8, 2), (3, 5, 7), (1, 64, 1000), (2, 40, 129), (9, 24, 300), (31, 72, 257), (33, 64, 128),
         (127, 65, 127), (128, 128, 128), (129, 136, 129), (300, 771, 501), (1000, 64, 80), (5000, 48, 17), (64, 96, 9001),
         (700, 1030, 333), (257, 192, 1024)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,d,v", SIZES)
def test_cross_entropy_and_gradients(n, d, v, dtype):
    h, w, t, up, _ = _data(n, d, v, dtype, seed=n * 7 + d * 3 + v, keep=0.8 if n > 2 else 1.0)
    out, gh, gw, tol, th, tw = _oracle(h, w, t=t, up=up)
    got = _ce(h, w, t, "none", up)
    _close(got[0], out, tol, "loss")
    _close(got[1], gh, th, "g_hidden")
    _close(got[2], gw, tw, "g_weight")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,d,v", SIZES)
def test_expected_center_and_gradients(n, d, v, dtype):
    h, w, _, up, c = _data(n, d, v, dtype, seed=n * 5 + d + v)
    out, gh, gw, tol, th, tw = _oracle(h, w, c=c, up=up)
    got = _ex(h, w, c, up)
    _close(got[0], out, tol, "depth")
    _close(got[1], gh, th, "g_hidden")
    _close(got[2], gw, tw, "g_weight")


@pytest.mark.gpu
@pytest.mark.parametrize("reduction", ["mean", "sum"])
@pytest.mark.parametrize("keep", [1.0, 0.5, 0.02])
def test_reductions(reduction, keep):
    n, d, v = 20000, 32, 50          # more rows than one listing workgroup takes
    h, w, t, _, _ = _data(n, d, v, torch.float32, seed=11, keep=keep)
    cnt = int((t != -100).sum())
    f = 1.0 / cnt if reduction == "mean" else 1.0
    up = torch.full((n,), f * 0.7, dtype=torch.float64, device=DEV)
    out, gh, gw, tol, th, tw = _oracle(h, w, t=t, up=up)
    got = _ce(h, w, t, reduction, torch.tensor(0.7, device=DEV))
    want = out.sum() * f
    _close(got[0], want, tol.sum() * f + 2.0 ** -23 * want.abs(), "loss")
    _close(got[1], gh, th + 2.0 ** -23 * gh.abs(), "g_hidden")      # the upstream value itself is 0.7 / count in float32
    _close(got[2], gw, tw + 2.0 ** -22 * gw.abs(), "g_weight")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_ignored_rows_are_not_read(dtype):
    """Features of ignored rows may be anything: NaN, infinities, the type's lowest value."""
    n, d, v = 300, 40, 70
    h, w, t, up, _ = _data(n, d, v, dtype, seed=3, keep=0.6)
    clean = _ce(h, w, t, "none", up)
    dirty = h.clone()
    ignored = (t == -100).nonzero()[:, 0]
    dirty[ignored[0::3]] = float("nan")
    dirty[ignored[1::3]] = float("inf")
    dirty[ignored[2::3]] = torch.finfo(dtype).min
    for a, b in zip(clean, _ce(dirty, w, t, "none", up)):
        assert torch.equal(a, b)
    assert torch.equal(clean[0][ignored], torch.zeros_like(clean[0][ignored]))
    assert torch.equal(clean[1][ignored], torch.zeros_like(clean[1][ignored]))


@pytest.mark.gpu
def test_nothing_left_and_bad_targets():
    h, w, t, up, _ = _data(40, 16, 10, torch.float32, seed=4)
    none = torch.full_like(t, -100)
    out, gh, gw = _ce(h, w, none, "mean")
    assert math.isnan(float(out)) and not gh.any() and not gw.any()
    out, gh, gw = _ce(h, w, none, "sum")
    assert float(out) == 0 and not gh.any() and not gw.any()
    out, gh, gw = _ce(h, w, none, "none", up)
    assert not out.any() and not gh.any() and not gw.any()
    bad = t.clone()
    bad[3], bad[7] = 10, -1                                     # classes are 0..9
    out, gh, gw = _ce(h, w, bad, "none", up)
    assert torch.isnan(out).nonzero()[:, 0].tolist() == [3, 7]
    assert torch.isnan(gh).any(1).nonzero()[:, 0].tolist() == [3, 7] and torch.isnan(gw).all()
    out, _, _ = _ce(h, w, t.where(t != 5, torch.full_like(t, 5)), "none", up, ignore=5)   # a real class may be the ignored one
    assert not out[t == 5].any() and (out[t != 5] > 0).all()


@pytest.mark.gpu
def test_no_rows():
    from depth_estimation_amd import metrics, synthesis
    w = torch.randn(6, 8, device=DEV, requires_grad=True)
    h = torch.randn(0, 8, device=DEV, requires_grad=True)
    t = torch.empty(0, dtype=torch.int64, device=DEV)
    assert math.isnan(float(metrics.linear_cross_entropy(h, w, t)))
    assert float(metrics.linear_cross_entropy(h, w, t, reduction="sum")) == 0
    out = metrics.linear_cross_entropy(h, w, t, reduction="none")
    assert out.shape == (0,)
    gh, gw = torch.autograd.grad(out.sum(), (h, w))
    assert gh.shape == (0, 8) and not gw.any()
    assert synthesis.depth_from_bins(h, w, torch.ones(6, device=DEV)).shape == (0,)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_layouts(dtype):
    """Strided, shifted, transposed, expanded and many-dimensional features give the bits of the plain layout."""
    from depth_estimation_amd import metrics, synthesis
    n, d, v = 60, 48, 30
    h, w, t, up, c = _data(n, d, v, dtype, seed=8, keep=0.9)
    base, exp = _ce(h, w, t, "none", up), _ex(h, w, c, up)
    wide = torch.zeros(n, d + 16, dtype=dtype, device=DEV)
    wide[:, 8:8 + d] = h
    shifted = torch.zeros(n * d + 1, dtype=dtype, device=DEV)
    shifted[1:] = h.reshape(-1)
    wsh = torch.zeros(v * d + 3, dtype=dtype, device=DEV)
    wsh[3:] = w.reshape(-1)
    odd = torch.zeros(n, d + 3, dtype=dtype, device=DEV)
    odd[:, 3:] = h
    forms = [(wide[:, 8:8 + d], w), (shifted[1:].view(n, d), wsh[3:].view(v, d)), (odd[:, 3:], w),
             (h.t().contiguous().t(), w.t().contiguous().t())]
    for hh, ww in forms:
        for a, b in zip(base, _ce(hh, ww, t, "none", up)):
            assert torch.equal(a, b)
        for a, b in zip(exp, _ex(hh, ww, c, up)):
            assert torch.equal(a, b)
    maps = h.view(3, 4, 5, d).permute(0, 3, 1, 2).contiguous().requires_grad_(True)     # (B,D,H,W) features of a network
    out = metrics.linear_cross_entropy(maps.permute(0, 2, 3, 1), w, t.view(3, 4, 5), reduction="none")
    assert torch.equal(out.detach().reshape(-1), base[0])
    (g,) = torch.autograd.grad(out, maps, up.view(3, 4, 5))
    assert torch.equal(g.permute(0, 2, 3, 1).reshape(n, d), base[1])
    one = h[:1].expand(n, d).requires_grad_(True)
    assert torch.equal(synthesis.depth_from_bins(one, w, c), exp[0][:1].expand(n))
    assert synthesis.depth_from_bins(h[0], w, c).shape == ()
    assert torch.equal(metrics.linear_cross_entropy(h, w, t.to(torch.int32), reduction="none"), base[0])


@pytest.mark.gpu
@pytest.mark.parametrize("scale_h,scale_w", [(1e-6, 1e6), (1e15, 1e-15), (1e-20, 1.0), (1e4, 1e-3)])
def test_float32_of_any_size(scale_h, scale_w):
    """The planes' scale follows the data: features and weights far from one lose nothing."""
    h, w, t, up, _ = _data(50, 33, 40, torch.float32, seed=9)
    h, w = h * scale_h, w * scale_w
    out, gh, gw, tol, th, tw = _oracle(h, w, t=t, up=up)
    got = _ce(h, w, t, "none", up)
    _close(got[0], out, tol, "loss")
    _close(got[1], gh, th, "g_hidden")
    _close(got[2], gw, tw, "g_weight")


@pytest.mark.gpu
@pytest.mark.parametrize("n,d,v", [(50, 33, 40), (200, 301, 700), (3, 40, 500)])
@pytest.mark.parametrize("scale_h,scale_w", [(1e-30, 1e30), (1e30, 1e-30), (2e37, 1e-37), (1e-36, 1e35), (1e-25, 1e-10), (1e-5, 1e-28)])
def test_float32_to_the_ends_of_its_range(n, d, v, scale_h, scale_w):
    """As above, to where float32's normal numbers end, in kernels for small heads, tiles and few rows."""
    h, w, t, up, c = _data(n, d, v, torch.float32, seed=n, keep=0.9 if n > 3 else 1.0)
    h, w = h * scale_h, w * scale_w
    for got, (out, gh, gw, tol, th, tw) in ((_ce(h, w, t, "none", up), _oracle(h, w, t=t, up=up)),
                                            (_ex(h, w, c, up), _oracle(h, w, c=c, up=up))):
        _close(got[0], out, tol, "output")
        for a, b, tol_ in ((got[1], gh, th), (got[2], gw, tw)):
            inside = b.abs() < torch.finfo(torch.float32).max / 4
            _close(a[inside], b[inside], tol_[inside], "gradient")


# factors of the upstream values and of the centres; float16's gradients stay in range only where one makes up for the other
FAR = [(torch.float32, 1e-36, 1.0), (torch.float32, 1e36, 1.0), (torch.bfloat16, 1e-28, 1.0), (torch.bfloat16, 1e36, 1.0)] + [
    (t, a, b) for t in TYPES for a, b in ((1e-30, 1e30), (1e30, 1e-30))]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,size_up,size_c", FAR, ids=str)
@pytest.mark.parametrize("n,d,v", [(60, 40, 50), (200, 64, 900)])
def test_upstreams_and_centers_of_any_size(n, d, v, dtype, size_up, size_c):
    h, w, t, up, c = _data(n, d, v, dtype, seed=n, keep=0.9)
    up, c = up * size_up, c * size_c
    pairs = [(_ex(h, w, c, up), _oracle(h, w, c=c, up=up))]
    if size_c == 1.0:
        pairs.append((_ce(h, w, t, "none", up), _oracle(h, w, t=t, up=up)))
        f = float(up[0])
        pairs.append((_ce(h, w, t, "sum", up[0]), _oracle(h, w, t=t, up=torch.full_like(up, f))))
    for got, (out, gh, gw, tol, th, tw) in pairs:
        if got[0].dim():
            _close(got[0], out, tol, "output")
        _close(got[1], gh, th, "g_hidden")
        _close(got[2], gw, tw, "g_weight")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_large_logits_and_upstreams(dtype):
    """Logits of +-100s, upstream values from 1e-6 to 1e6 and zero in one call."""
    h, w, t, up, _ = _data(200, 32, 60, dtype, seed=10, spread=60.0)
    up = up * (10.0 ** torch.linspace(-6, 6, 200, device=DEV))
    up[17] = 0
    out, gh, gw, tol, th, tw = _oracle(h, w, t=t, up=up)
    fit = torch.finfo(dtype).max
    got = _ce(h, w, t, "none", up)
    _close(got[0], out, tol, "loss")
    for a, b, tol_ in ((got[1], gh, th), (got[2], gw, tw)):
        inside = b.abs() < fit / 2
        _close(a[inside], b[inside], tol_[inside], "gradient")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,d,v", [(1, 37, 1001), (3, 40, 500), (4, 250, 60), (20, 70, 500), (60, 40, 50), (200, 64, 900),
                                   (2500, 301, 4100), (1500, 96, 20000)])
def test_huge_logits_give_whole_probabilities(n, d, v, dtype):
    """Logits of 1e9 (float16: 1e5): the backward's are the forward's bit by bit, so a probability is 1 or 0 however large their
    rounding is.  Rows whose two largest logits lie within what that may be are left out (their upstream is 0), and so is dl's
    error: dl is 0 or +-upstream, rounded to its stored type."""
    h, w, t, up, c = _data(n, d, v, dtype, seed=n + v)
    h = (h.float() * (2.0 ** 11 if dtype == torch.float16 else 2.0 ** 28)).to(dtype)
    l = h.double() @ w.double().T
    two = l.topk(2, dim=1).values
    far = two[:, 0] - two[:, 1] > 40 + 2.0 ** -20 * d * (h.double().abs() @ w.double().abs().T).max(dim=1).values / d ** 0.5
    assert bool(far.any())
    up = torch.where(far, up, torch.zeros_like(up))
    p = torch.nn.functional.one_hot(l.argmax(1), v).double()
    u = 2.0 ** -21 if dtype == torch.float32 else U[dtype]
    pairs = [(_ce(h, w, t, "none", up), (p - torch.nn.functional.one_hot(t, v)) * up.double()[:, None]),
             (_ex(h, w, c, up), torch.zeros_like(p))]
    for got, dl in pairs:
        gh, gw = dl @ w.double(), dl.T @ h.double()
        # a probability of exp(-40) and less beside: 4e-18 of the upstream (times the largest centre)
        err = (u + (n + v + 8) * 2.0 ** -24) * dl.abs() + 1e-15 * up.double()[:, None] * (1.0 + 80.0)
        split = 2.0 ** -21 if dtype == torch.float32 else 0.0
        _close(got[1], gh, (err + split * dl.abs()) @ w.double().abs() + U[dtype] * gh.abs() + 2.0 ** -24, "g_hidden")
        inside = gw.abs() < torch.finfo(dtype).max / 2
        tw = (err + split * dl.abs()).T @ h.double().abs() + U[dtype] * gw.abs() + 2.0 ** -24
        _close(got[2][inside], gw[inside], tw[inside], "g_weight")
    assert torch.equal(pairs[1][0][0][far], c[l.argmax(1)][far])


def _row_oracle(h, w, up, t=None, c=None):
    """g_hidden and its tolerance row by row: a row's gradient is its upstream value times what it is for 1, and so is what it may be
    off by, whatever the other rows' upstream"""
    one = torch.ones_like(up)
    _, gh, _, _, th, _ = _oracle(h, w, t=t, c=c, up=one)
    sub = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}[h.dtype]
    s = up.double()[:, None]
    return gh * s, th * s.abs() + sub


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,d,v", [(3, 40, 500), (60, 40, 50), (70, 33, 50), (200, 64, 900), (9000, 24, 40), (3000, 136, 1500),
                                   (700, 131, 2500), (6000, 256, 700), (1500, 24, 200_001)])
def test_a_row_keeps_its_gradient_beside_larger_ones(n, d, v, dtype):
    """Upstream values that span 2^26 (float16: as far as its results reach), 2^80 and zero: every row's own digits, and dW's as
    far as they follow from the largest."""
    lo, hi = (-3.0, 4.5) if dtype == torch.float16 else (-20.0, 4.0)
    h, w, t, up, c = _data(n, d, v, dtype, seed=n + d)
    c = c / 80
    g = torch.Generator().manual_seed(n)
    up = up * (10.0 ** (lo + (hi - lo) * torch.rand(n, generator=g))).to(DEV)
    up[n // 2] = 0
    if n > 3:
        t[1::7] = -100
    if v > 100_000:          # pieces of the classes, and their sums: the oracle takes every 13th row
        pick = torch.arange(0, n, 13, device=DEV)
    else:
        pick = torch.arange(n, device=DEV)
    for ce in (True, False):
        k = dict(t=t) if ce else dict(c=c)
        got = _ce(h, w, t, "none", up) if ce else _ex(h, w, c, up)
        gh, th = _row_oracle(h[pick], w, up[pick], t=t[pick] if ce else None, c=None if ce else c)
        fits = gh.abs() < torch.finfo(dtype).max / 2
        mine = got[1][pick]
        _close(torch.where(fits, mine.double(), 0.0), torch.where(fits, gh, 0.0), th, "g_hidden")
        big = (gh.abs() > th) & fits
        assert not (mine == 0)[big].any()
        if v <= 100_000:
            _, _, gw, _, _, tw = _oracle(h, w, up=up, **k)
            fits = gw.abs() < torch.finfo(dtype).max / 2
            _close(got[2][fits], gw[fits], tw[fits], "g_weight")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,d,v", [(60, 40, 50), (200, 64, 900), (500, 131, 700)])
def test_weighted_out_rows_leave_no_trace(n, d, v, dtype):
    """Rows of large features and zero upstream (a caller's own mask): dW is that of the other rows, as exactly."""
    h, w, t, up, c = _data(n, d, v, dtype, seed=n + v)
    small = h * 2.0 ** -9
    loud = small.clone()
    loud[::5] = h[::5] * 2.0 ** 5
    up[::5] = 0
    quiet = small.clone()
    quiet[::5] = 0
    for a, b, want in ((_ce(loud, w, t, "none", up), _ce(quiet, w, t, "none", up), _oracle(quiet, w, t=t, up=up)),
                       (_ex(loud, w, c, up), _ex(quiet, w, c, up), _oracle(quiet, w, c=c, up=up))):
        _close(a[2], want[2], want[5], "g_weight")
        _close(b[2], want[2], want[5], "g_weight")
        assert not a[1][::5].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("kind", ["log", "far", "negative", "mixed"])
@pytest.mark.parametrize("n,d,v", [(4, 40, 500), (60, 40, 50), (200, 64, 900), (9000, 24, 40), (3000, 136, 1500)])
def test_small_depths_beside_large_centers(n, d, v, kind, dtype):
    """Centres over nine decades, or a last one of 1e12: rows that are sure of small ones keep their gradient's digits.  p (c - E) is
    rounded relative to sum p |c| (centres of one sign) or, where signs differ, to the largest centre."""
    g = torch.Generator().manual_seed(n + v)
    w = (torch.randn(v, d, generator=g) / math.sqrt(d)).to(dtype).to(DEV)
    cls = torch.randint(0, v - 1, (n,), generator=g)
    h = (torch.randn(n, d, generator=g) + 8.0 * w.float().cpu()[cls] * math.sqrt(d / 8)).to(dtype).to(DEV)
    c = torch.logspace(-6, 3, v).to(DEV)
    if kind == "far":
        w[-1] = -8 * h.float().mean(0).to(dtype) - 4 * w.abs().amax()
        c = torch.linspace(1.0, 2.0, v).to(DEV)
        c[-1] = 1e12
        h = torch.cat([h[:, :-1].abs(), h[:, -1:].abs()], 1)       # the far class is out of reach: features and weight disagree
        w[-1] = -(60.0 / h.float().sum(1).min()).clamp(min=1.0).to(dtype) * 2
    if kind == "negative":
        c = -c
    if kind == "mixed":
        c = c - 1e-4
    up = (torch.rand(n, generator=g) + 0.5).to(DEV)
    got = _ex(h, w, c, up)
    H, W, C, U64 = h.double(), w.double(), c.double(), up.double()[:, None]
    p = torch.softmax(H @ W.T, 1)
    E = (p @ C)[:, None]
    size = p @ C.abs()
    split = 2.0 ** -21 if dtype == torch.float32 else 0.0
    el = (split + (d + 4) * 2.0 ** -24) * (H.abs() @ W.abs().T)
    ep = 2 * el.max(dim=1, keepdim=True).values + (v + 32) * 2.0 ** -24
    tol = (ep[:, 0] * size) + 4 * 2.0 ** -24 * size
    dl = p * (C[None] - E) * U64
    ref = C.abs().max() if kind == "mixed" else size[:, None]
    u = {torch.float32: 2.0 ** -21, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
    err = (p * (ep * (C[None] - E).abs() + tol[:, None] + 2.0 ** -23 * C.abs()[None])) * U64 + u * dl.abs()
    if dtype != torch.bfloat16:
        err = err + 2.0 ** -37 * ref * U64
    out = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
    sub = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}[dtype]
    _close(got[0], E[:, 0], tol, "depth")
    gh = dl @ W
    fits = gh.abs() < torch.finfo(dtype).max / 2
    th = (err + (split + (v + 8) * 2.0 ** -24) * dl.abs()) @ W.abs() + out * gh.abs() + sub
    _close(torch.where(fits, got[1].double(), 0), torch.where(fits, gh, 0), th, "g_hidden")
    gw = dl.T @ H
    if dtype != torch.bfloat16 and kind != "mixed":      # dW is relative to the row that reaches farthest
        err = err + 2.0 ** -37 * (size[:, None] * U64).max()
    tw = (err + (split + (n + 8) * 2.0 ** -24) * dl.abs()).T @ H.abs() + out * gw.abs() + sub
    fits = gw.abs() < torch.finfo(dtype).max / 2
    _close(torch.where(fits, got[2].double(), 0), torch.where(fits, gw, 0), tw, "g_weight")


@pytest.mark.gpu
@pytest.mark.parametrize("reduction", ["none", "mean"])
@pytest.mark.parametrize("n,d,v", [(20, 70, 500), (60, 40, 50), (200, 64, 900), (300, 515, 70), (9000, 24, 40), (3000, 136, 1500)])
def test_float32_rows_do_not_see_each_other(n, d, v, reduction):
    """Features of 1e-12, 1 and 1e12 in the rows of one batch: a row's loss, depth and gradient have the bits that they have in a
    batch of its like (the same sizes, so the same kernels), and dW what follows from the largest."""
    h, w, t, up, c = _data(n, d, v, torch.float32, seed=n + d)
    size = torch.ones(n, device=DEV)
    size[0::4], size[1::4], size[2::4] = 1e12, 1e-12, 1e30
    if reduction == "mean":          # a count that every batch has
        up = torch.full_like(up, 0.5)
    mixed = h * size[:, None]
    for f in (1.0, 1e12, 1e-12, 1e30):
        rows = size == f
        if not bool(rows.any()):
            continue
        alike = h * f
        a, b = _ce(mixed, w, t, "none", up), _ce(alike, w, t, "none", up)
        assert torch.equal(a[0][rows], b[0][rows]) and torch.equal(a[1][rows], b[1][rows])
        a, b = _ex(mixed, w, c, up), _ex(alike, w, c, up)
        assert torch.equal(a[0][rows], b[0][rows]) and torch.equal(a[1][rows], b[1][rows])
    size[2::4] = 1e-6
    mixed = h * size[:, None]
    scale = torch.tensor(0.5 * n, device=DEV)
    got = _ce(mixed, w, t, reduction, up if reduction == "none" else scale)
    out, gh, gw, tol, th, tw = _oracle(mixed, w, t=t, up=up if reduction == "none" else torch.full_like(up, 0.5))
    row = (2.0 ** -21 + (d + 4) * 2.0 ** -24) * (mixed.double().abs() @ w.double().abs().T)
    row = row.max(dim=1).values + 2.0 ** -39 * d * mixed.double().abs().max(dim=1).values * w.double().abs().max()
    own = 2 * row + (v + 32) * 2.0 ** -24 + 4 * 2.0 ** -24 * ((mixed.double() @ w.double().T).abs().max(dim=1).values + out.abs() + 1)
    if reduction == "none":
        _close(got[0], out, own, "loss")
    _close(got[1], gh, th, "g_hidden")
    _close(got[2], gw, tw + (2.0 ** -22 * gw.abs() if reduction == "mean" else 0.0), "g_weight")


@pytest.mark.gpu
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
@pytest.mark.parametrize("n,d,v", [(4, 40, 500), (60, 40, 50), (200, 64, 900)])
def test_float32_rows_of_zeros_and_of_masked_size(n, d, v, reduction):
    """Rows of zeros, and rows of 1e35 with zero upstream or ignored: the gradient of the weight is that without them."""
    h, w, t, up, c = _data(n, d, v, torch.float32, seed=n)
    h = h * 1e-3
    h[0], h[n // 2] = 0, 0
    loud = h.clone()
    loud[1::3] = 1e32 * h[1::3]
    if reduction == "none":
        up[1::3] = 0
        pairs = [(_ce(loud, w, t, "none", up), _oracle(torch.where((up == 0)[:, None], 0.0, h), w, t=t, up=up)),
                 (_ex(loud, w, c, up), _oracle(torch.where((up == 0)[:, None], 0.0, h), w, c=c, up=up))]
    else:
        t[1::3] = -100
        f = 1.0 / int((t != -100).sum()) if reduction == "mean" else 1.0
        pairs = [(_ce(loud, w, t, reduction), _oracle(h, w, t=t, up=torch.full((n,), f, dtype=torch.float64, device=DEV)))]
    for got, (_, gh, gw, _, th, tw) in pairs:
        _close(got[2], gw, tw + 2.0 ** -22 * gw.abs(), "g_weight")
        quiet = torch.arange(n, device=DEV) % 3 != 1
        _close(got[1][quiet], gh[quiet], (th + 2.0 ** -22 * gh.abs())[quiet], "g_hidden")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_confident_rows(dtype):
    """Rows that are all but certain of their class: p - 1 keeps its digits, nothing overflows."""
    n, d, v = 64, 64, 64
    w = torch.eye(v, d, device=DEV).to(dtype)
    h = (40 * torch.eye(n, d, device=DEV)).to(dtype)
    t = torch.arange(n, device=DEV)
    up = torch.ones(n, device=DEV)
    out, gh, gw, tol, th, tw = _oracle(h, w, t=t, up=up)
    got = _ce(h, w, t, "none", up)
    _close(got[0], out, tol, "loss")
    _close(got[1], gh, th, "g_hidden")
    _close(got[2], gw, tw, "g_weight")


@pytest.mark.gpu
def test_pieces_of_the_classes_join():
    """More rows times classes than one piece of dl holds: the gradient of the features adds up over pieces."""
    n, d, v = 40000, 24, 5000          # 2 bytes x 40000 rows: 3328 classes a piece
    h, w, t, up, _ = _data(n, d, v, torch.bfloat16, seed=12, keep=0.9)
    got = _ce(h, w, t, "none", up)
    pick = torch.arange(0, n, 997, device=DEV)
    out, gh, _, tol, th, _ = _oracle(h[pick], w, t=t[pick], up=up[pick])
    _close(got[0][pick], out, tol, "loss")
    _close(got[1][pick], gh, th, "g_hidden")
    gw = torch.zeros(v, d, dtype=torch.float64, device=DEV)
    tw = torch.zeros_like(gw)
    for lo in range(0, n, 4000):
        s = slice(lo, lo + 4000)
        _, _, g, _, _, tt = _oracle(h[s], w, t=t[s], up=up[s])
        gw, tw = gw + g, tw + tt
    _close(got[2], gw, tw + n * 2.0 ** -24 * tw + U[torch.bfloat16] * gw.abs(), "g_weight")


@pytest.mark.gpu
def test_gradient_is_the_difference_quotient():
    n, d, v = 6, 10, 9
    h, w, t, up, c = _data(n, d, v, torch.float32, seed=13)
    from depth_estimation_amd import metrics, synthesis
    g = torch.Generator().manual_seed(1)
    dh, dw = torch.randn(n, d, generator=g).to(DEV), torch.randn(v, d, generator=g).to(DEV)
    for f, (_, gh, gw) in ((lambda a, b: metrics.linear_cross_entropy(a, b, t, reduction="none"), _ce(h, w, t, "none", up)),
                           (lambda a, b: synthesis.depth_from_bins(a, b, c), _ex(h, w, c, up))):
        e = 2.0 ** -7
        quotient = ((f(h + e * dh, w + e * dw) - f(h - e * dh, w - e * dw)).double() * up.double()).sum() / (2 * e)
        slope = (gh.double() * dh).sum() + (gw.double() * dw).sum()
        # third derivatives of order 100 times e^2 / 6, and float32 outputs of size 80 over 2 e
        assert abs(float(quotient - slope)) <= 0.02 * abs(float(slope)) + 0.02


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_same_bits_every_time(dtype):
    h, w, t, up, c = _data(3000, 64, 700, dtype, seed=14, keep=0.7)
    a, b = _ce(h, w, t, "mean"), _ce(h, w, t, "mean")
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    a, b = _ex(h, w, c, up), _ex(h, w, c, up)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.gpu
def test_one_gradient_alone_and_frozen_inputs():
    from depth_estimation_amd import metrics
    h, w, t, up, _ = _data(70, 32, 20, torch.bfloat16, seed=15)
    _, gh, gw = _ce(h, w, t, "none", up)
    h1 = h.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(metrics.linear_cross_entropy(h1, w, t, reduction="none"), h1, up)[0], gh)
    w1 = w.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(metrics.linear_cross_entropy(h, w1, t, reduction="none"), w1, up)[0], gw)
    assert not metrics.linear_cross_entropy(h, w, t).requires_grad
    out = metrics.linear_cross_entropy(h1, w1, t)
    (g,) = torch.autograd.grad(out, h1, create_graph=True, retain_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()


@pytest.mark.gpu
def test_streams_and_captured_graphs():
    """Another stream; two graphs captured one after the other and replayed in turn with eager calls between."""
    from depth_estimation_amd import metrics, synthesis
    h, w, t, up, c = _data(500, 64, 200, torch.bfloat16, seed=16, keep=0.8)
    want, wexp = _ce(h, w, t, "mean"), _ex(h, w, c, up)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = _ce(h, w, t, "mean")
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))

    def capture(f):
        with torch.cuda.stream(s):
            f()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = f()
        return g, out

    h2, t2 = h.clone(), t.clone()
    g1, o1 = capture(lambda: _ce(h2, w, t2, "mean"))
    g2, o2 = capture(lambda: _ex(h2, w, c, up))
    other, _, tother, _, _ = _data(500, 64, 200, torch.bfloat16, seed=17, keep=0.5)
    for k in range(4):
        src, ts = (h, t) if k % 2 == 0 else (other, tother)
        h2.copy_(src)
        t2.copy_(ts)
        torch.cuda.synchronize()
        g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        e1, e2 = _ce(src, w, ts, "mean"), _ex(src, w, c, up)
        assert all(torch.equal(a, b) for a, b in zip(o1, e1))
        assert all(torch.equal(a, b) for a, b in zip(o2, e2))
    assert all(torch.equal(a, b) for a, b in zip(_ex(h, w, c, up), wexp))
    del g1, g2, o1, o2
    assert torch.isfinite(metrics.linear_cross_entropy(h, w, t)) and torch.isfinite(synthesis.depth_from_bins(h, w, c)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,d,v", [(3, 40, 500), (60, 40, 50), (200, 64, 900), (9000, 72, 600)])
def test_captured_with_upstreams_that_change(n, d, v, dtype):
    """Row scales are found anew in every replay: features and upstream values of another size, other rows left out, eager calls
    between."""
    h, w, t, up, c = _data(n, d, v, dtype, seed=n, keep=0.8 if n > 3 else 1.0)
    h2, t2, up2 = h.clone(), t.clone(), up.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _ce(h2, w, t2, "none", up2), _ex(h2, w, c, up2), _ce(h2, w, t2, "mean")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = _ce(h2, w, t2, "none", up2) + _ex(h2, w, c, up2) + _ce(h2, w, t2, "mean")
    for k in range(4):
        spread = 10.0 ** (torch.arange(n, device=DEV) % (2 + k) - 1.0)
        h2.copy_(h * (1.0, 0.25, 1.0, 2.0 ** -6)[k])
        up2.copy_(up * spread * (1.0, 1e-2, 1.0, 30.0)[k])
        t2.copy_(t if k % 2 == 0 else t.flip(0))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        eager = _ce(h2, w, t2, "none", up2) + _ex(h2, w, c, up2) + _ce(h2, w, t2, "mean")
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


@pytest.mark.gpu
def test_head_into_the_photometric_loss():
    """The operators together, as a trainer uses them: features -> expected depth -> warp and photometric loss, plus the cross
    entropy of the same head where a depth was measured; one backward, one orthogonalised step.  Checked: the head's gradient
    equals the chain of its parts."""
    import depth_estimation_amd as de
    B, S, H, W, D, V = 1, 2, 24, 80, 32, 40
    g = torch.Generator().manual_seed(2)
    feats = torch.randn(B, S, H, W, D, generator=g).to(DEV).requires_grad_(True)
    weight = (0.3 * torch.randn(V, D, generator=g)).to(DEV).requires_grad_(True)
    centers = torch.logspace(0, 1.9, V, device=DEV)
    src, tgt = torch.rand(B, S, 3, H, W, generator=g).to(DEV), torch.rand(B, 3, H, W, generator=g).to(DEV)
    K, Kinv = de.fused.intrinsics(W, H, DEV)
    pose = de.synthesis.construct_pose_batch(0.01 * torch.randn(B * S, 6, generator=g).to(DEV)).reshape(B, S, 3, 4)
    measured = torch.randint(0, V, (B, S, H, W), generator=g)
    measured[torch.rand(B, S, H, W, generator=g) < 0.9] = -100
    measured = measured.to(DEV)
    depth = de.synthesis.depth_from_bins(feats, weight, centers)
    photo = de.fused.train_step_loss(src, tgt, depth.unsqueeze(2), pose, K, Kinv)["total"]
    ce = de.metrics.linear_cross_entropy(feats, weight, measured)
    gf, gw = torch.autograd.grad(photo + 0.1 * ce, (feats, weight))
    d = depth.detach().requires_grad_(True)
    (gd,) = torch.autograd.grad(de.fused.train_step_loss(src, tgt, d.unsqueeze(2), pose, K, Kinv)["total"], d)
    flat = feats.detach().reshape(-1, D)
    _, eh, ew, _, teh, tew = _oracle(flat, weight.detach(), c=centers, up=gd.reshape(-1))
    cnt = int((measured != -100).sum())
    t = measured.reshape(-1)
    _, ch, cw, _, tch, tcw = _oracle(flat, weight.detach(), t=t, up=torch.full((len(t),), 0.1 / cnt, device=DEV,
                                                                              dtype=torch.float64))
    _close(gf.reshape(-1, D), eh + ch, teh + tch + 2.0 ** -22 * (eh.abs() + ch.abs()), "g_hidden")
    _close(gw, ew + cw, tew + tcw + 2.0 ** -22 * (ew.abs() + cw.abs()), "g_weight")
    before = weight.detach().clone()
    weight.grad = gw
    de.optim.Muon([weight], lr=0.1, momentum=0.9).step()
    step = (before - weight.detach()) / 0.1 / max(1.0, V / D) ** 0.5
    assert torch.allclose(step, de.optim.orthogonalize(gw * 1.9), rtol=0, atol=1e-4)


# ------------------------------------------------------------------------------------------------------- refusals
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,d,v", [(2500, 301, 4100), (60000, 504, 520), (3000, 500, 9000)])
def test_large_tiles(n, d, v, dtype):
    """Sizes whose products take tiles of 256 x 256, whole and across edges, with the sums over classes and over rows split."""
    h, w, t, up, c = _data(n, d, v, dtype, seed=n + d + v, keep=0.9)
    for got, (out, gh, gw, tol, th, tw) in ((_ce(h, w, t, "none", up), _oracle(h, w, t=t, up=up)),
                                            (_ex(h, w, c, up), _oracle(h, w, c=c, up=up))):
        _close(got[0], out, tol, "output")
        _close(got[1], gh, th, "g_hidden")
        _close(got[2], gw, tw, "g_weight")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_pieces_with_a_row_of_nan(dtype):
    """70001 classes in two pieces (three in float32), the sum over them split.  A row of NaN gradients reaches no other row."""
    n, d, v, bad = 3000, 500, 70001, 1501
    h, w, t, up, _ = _data(n, d, v, dtype, seed=21)
    t[7] = v - 1                                   # a target in the last piece
    pick = torch.arange(bad - 40, bad + 40, device=DEV)
    out, gh, _, tol, th, _ = _oracle(h[pick], w, t=t[pick], up=up[pick])
    # the scale of dl follows the largest upstream of all rows: its rounding floor with it
    th = th * (1.0 if dtype == torch.bfloat16 else float(up.max() / up[pick].max()))
    t[bad] = v + 5
    got = _ce(h, w, t, "none", up)
    keep = pick != bad
    _close(got[0][pick][keep], out[keep], tol[keep], "loss")
    _close(got[1][pick][keep], gh[keep], th[keep], "g_hidden")
    assert torch.isnan(got[0][bad]) and torch.isnan(got[1][bad]).all() and torch.isnan(got[2]).all()
    assert torch.isfinite(got[1][torch.arange(n, device=DEV) != bad]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("n,d,v", [(400, 64, 8), (777, 250, 128), (600, 120, 288), (3000, 64, 80), (500, 33, 289), (1, 56, 3784),
                                   (2, 40, 500), (4, 250, 2000), (25, 1744, 1001), (483, 56, 19229), (5719, 64, 1232), (300, 515, 700),
                                   (3000, 96, 7000)])
def test_smaller_heads_round_once(n, d, v, dtype):
    """16-bit heads of up to 2^31 products, on chip those of few rows a class: as float32 heads of the same values, and rounded once.
    The logits' gradient is held in two planes, 2^-16 (bfloat16) of it or less is dropped."""
    h, w, t, up, c = _data(n, d, v, dtype, seed=n + d + v, keep=0.8)
    for got, k in ((_ce(h, w, t, "none", up), dict(t=t)), (_ex(h, w, c, up), dict(c=c))):
        _, gh, gw, _, th, tw = _oracle(h.float(), w.float(), up=up, **k)
        p = torch.softmax(h.double() @ w.double().T, 1)
        if "t" in k:
            dl = (p + torch.nn.functional.one_hot(t.clamp(min=0), v)) * (up * (t != -100)).double()[:, None]
        else:
            dl = p * (c.double()[None] - (p @ c.double())[:, None]).abs() * up.double()[:, None]
        sub = 2.0 ** -24 if dtype == torch.float16 else 2.0 ** -133
        _close(got[1], gh, th + 2.0 ** -16 * dl @ w.double().abs() + U[dtype] * gh.abs() + sub, "g_hidden")
        live = torch.ones(n, dtype=torch.bool, device=DEV) if "c" in k else t != -100
        _close(got[2], gw, tw + 2.0 ** -16 * dl.T @ torch.where(live[:, None], h, 0).double().abs() + U[dtype] * gw.abs() + sub,
               "g_weight")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_several_pieces_with_rows_left_out(dtype):
    """70001 classes of 4000 rows: two pieces (four in float32), a smaller last one, rows left out, targets at the pieces' ends.  Cross
    entropy and the expectation, whose centres belong to the piece; every row and every class checked."""
    n, d, v = 4000, 40, 70001
    h, w, t, up, c = _data(n, d, v, dtype, seed=41, keep=0.8)
    for k, cls in enumerate((v - 1, 0, 17535, 17536, 35007, 35008, 52608, 70000)):
        t[10 + k] = cls
    for got, k in ((_ce(h, w, t, "none", up), dict(t=t)), (_ex(h, w, c, up), dict(c=c))):
        out, gh, gw, tol, th, tw = _oracle(h, w, up=up, **k)
        _close(got[0], out, tol, "output")
        _close(got[1], gh, th, "g_hidden")
        _close(got[2], gw, tw, "g_weight")
        del out, gh, gw, tol, th, tw


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,d,v,keep", [(515, 96, 15593, 0.9), (914, 131, 43010, 0.9), (227, 131, 3165, 0.9), (121, 96, 3187, 1.0),
                                        (16961, 96, 753, 0.9), (1706, 131, 38516, 0.9), (16593, 96, 791, 0.05),
                                        (60000, 504, 520, 0.02), (60000, 504, 520, 0.0)])
def test_sums_with_splits_that_get_nothing(n, d, v, keep, dtype):
    """Sums over classes whose steps of 64 are no multiple of the splits (the last ones, up to nine of 128, are empty), in tiles of
    every size, and sums over rows most of which are left out, so that most splits are."""
    h, w, t, up, _ = _data(n, d, v, dtype, seed=n + v, keep=keep)
    out, gh, gw, tol, th, tw = _oracle(h, w, t=t, up=up)
    got = _ce(h, w, t, "none", up)
    _close(got[0], out, tol, "loss")
    _close(got[1], gh, th, "g_hidden")
    _close(got[2], gw, tw, "g_weight")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,d,v", [(777, 250, 128), (600, 120, 288), (900, 64, 576), (500, 33, 289), (400, 256, 64), (300, 128, 144)])
def test_small_heads_up_to_what_fits(n, d, v, dtype):
    """Heads around the largest weights that are held on chip; the loss of another forward replayed from a captured graph."""
    h, w, t, up, c = _data(n, d, v, dtype, seed=n + d + v, keep=0.7)
    for got, (out, gh, gw, tol, th, tw) in ((_ce(h, w, t, "none", up), _oracle(h, w, t=t, up=up)),
                                            (_ex(h, w, c, up), _oracle(h, w, c=c, up=up))):
        _close(got[0], out, tol, "output")
        _close(got[1], gh, th, "g_hidden")
        _close(got[2], gw, tw, "g_weight")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    x = h.clone()
    with torch.cuda.stream(s):
        _ex(x, w, c, up)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = _ex(x, w, c, up)
    for k in (1.0, 0.5, 2.0):
        x.copy_(h * k)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, _ex(x, w, c, up)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 7, 8, 9, 32, 33])
def test_few_rows(n, dtype):
    """Every number of rows around those that have kernels of their own, against many classes; two backward passes of one
    forward give the same bits."""
    from depth_estimation_amd import metrics, synthesis
    for d, v in ((37, 1001), (1300, 700), (10300, 33)):
        h, w, t, up, c = _data(n, d, v, dtype, seed=n + d, keep=1.0)
        if n > 2:
            t[1] = -100
        hg, wg = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
        for out, want in ((metrics.linear_cross_entropy(hg, wg, t, reduction="none"), _oracle(h, w, t=t, up=up)),
                          (synthesis.depth_from_bins(hg, wg, c), _oracle(h, w, c=c, up=up))):
            first = torch.autograd.grad(out, (hg, wg), up, retain_graph=True)
            again = torch.autograd.grad(out, (hg, wg), up)
            assert all(torch.equal(a, b) for a, b in zip(first, again))
            _close(out.detach(), want[0], want[3], "output")
            _close(first[0], want[1], want[4], "g_hidden")
            _close(first[1], want[2], want[5], "g_weight")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,d,v", [(1, 64, 16384), (8, 37, 16000), (32, 72, 16001), (16, 40, 15999), (32, 200, 17000)])
def test_few_rows_of_many_classes(n, d, v, dtype):
    """Around where up to 32 rows take a shape of their own."""
    h, w, t, up, c = _data(n, d, v, dtype, seed=n + v, keep=0.8 if n > 1 else 1.0)
    for got, (out, gh, gw, tol, th, tw) in ((_ce(h, w, t, "none", up), _oracle(h, w, t=t, up=up)),
                                            (_ex(h, w, c, up), _oracle(h, w, c=c, up=up))):
        _close(got[0], out, tol, "output")
        _close(got[1], gh, th, "g_hidden")
        _close(got[2], gw, tw, "g_weight")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,d,v", [(6143, 64, 560), (6144, 64, 560), (6500, 120, 288), (6500, 250, 128), (6200, 33, 289)])
def test_heads_on_chip_with_large_weights(n, d, v, dtype):
    """Around where a head whose weight takes more than 40 KB is held on chip."""
    h, w, t, up, c = _data(n, d, v, dtype, seed=n + v, keep=0.7)
    for got, (out, gh, gw, tol, th, tw) in ((_ce(h, w, t, "none", up), _oracle(h, w, t=t, up=up)),
                                            (_ex(h, w, c, up), _oracle(h, w, c=c, up=up))):
        _close(got[0], out, tol, "output")
        _close(got[1], gh, th, "g_hidden")
        _close(got[2], gw, tw, "g_weight")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 33, 300])
def test_answers_without_gradients(n, dtype):
    """What a program that only answers gets: few rows of a weight that would have to be packed have kernels of their own."""
    from depth_estimation_amd import metrics, synthesis
    for d, v in ((37, 1001), (256, 700), (1300, 80), (10300, 33)):
        h, w, t, up, c = _data(n, d, v, dtype, seed=n + d)
        if n > 2:
            t[1] = -100
        out, _, _, tol, _, _ = _oracle(h, w, t=t, up=up)
        _close(metrics.linear_cross_entropy(h, w, t, reduction="none"), out, tol, "loss")
        total = out.sum()
        _close(metrics.linear_cross_entropy(h, w, t, reduction="sum"), total, tol.sum() + 2.0 ** -23 * total.abs(), "sum")
        exp, _, _, etol, _, _ = _oracle(h, w, c=c, up=up)
        depth = synthesis.depth_from_bins(h, w, c)
        _close(depth, exp, etol, "depth")
        assert not depth.requires_grad
        with torch.no_grad():
            assert torch.equal(synthesis.depth_from_bins(h.clone().requires_grad_(True), w, c), depth)
        _close(synthesis.depth_from_bins(h.clone().requires_grad_(True), w, c).detach(), exp, etol, "depth, with a gradient")


@pytest.mark.gpu
def test_rows_far_apart():
    """A row pitch of ten million bytes: 250 rows lie across more than 2^31 bytes."""
    from depth_estimation_amd import synthesis
    n, d, v = 250, 64, 700
    h, w, t, up, c = _data(n, d, v, torch.bfloat16, seed=23)
    far = torch.empty(n, 5_000_000, dtype=torch.bfloat16, device=DEV)[:, :d]
    far.copy_(h)
    for a, b in zip(_ex(far, w, c, up), _ex(h, w, c, up)):
        assert torch.equal(a, b)
    for a, b in zip(_ce(far, w, t, "none", up), _ce(h, w, t, "none", up)):
        assert torch.equal(a, b)
    assert torch.equal(synthesis.depth_from_bins(far, w[:40], c[:40]), synthesis.depth_from_bins(h, w[:40], c[:40]))


@pytest.mark.gpu
def test_two_calls_at_once():
    """Calls of different inputs under way on two streams."""
    a, b = (_data(2000, 72, 600, torch.float32, seed=k, keep=0.8) for k in (31, 32))
    want = [(_ce(h, w, t, "mean"), _ex(h, w, c, up)) for h, w, t, up, c in (a, b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for k, (h, w, t, up, c) in enumerate((a, b)):
            with torch.cuda.stream(streams[k]):
                got[k].append((_ce(h, w, t, "mean"), _ex(h, w, c, up)))
    torch.cuda.synchronize()
    for k in (0, 1):
        for ce, ex in got[k]:
            assert all(torch.equal(x, y) for x, y in zip(ce + ex, want[k][0] + want[k][1]))


def test_refusals_of_answers_on_the_host():
    """Every wrong argument of the C entries of a forward alone, before any launch."""
    from depth_estimation_amd import _lib as L
    if not os.path.exists(L.LIB_PATH):
        pytest.skip("libdepthsynth.so not built (run __graft_entry__.build())")
    lib, fake, big = L.lib(), 0x1000, 1 << 40

    def ce(h=fake, ldh=64, w=fake, t=fake, dt=2, n=8, d=64, v=16, red=2, out=fake, ws=fake, nb=big):
        return lib.ds_linear_ce_eval(h, ldh, w, t, dt, n, d, v, -100, red, out, ws, nb, None)

    def ex(h=fake, w=fake, c=fake, dt=2, n=8, out=fake, ws=fake, nb=big):
        return lib.ds_bin_expect_eval(h, 64, w, c, dt, n, 64, 16, out, ws, nb, None)

    for rc, want in [(ce(h=None), -1), (ce(w=None), -1), (ce(t=None), -1), (ce(out=None), -1), (ce(n=0), -1), (ce(ldh=63), -1),
                     (ce(red=3), -1), (ce(dt=3), -2), (ce(n=(1 << 24) + 1), -2), (ce(ws=None), -3), (ce(nb=64), -3),
                     (ce(ws=fake + 4), -3), (ce(w=fake + 2), -1), (ex(h=None), -1), (ex(c=None), -1), (ex(out=None), -1), (ex(n=0), -1),
                     (ex(dt=9), -2), (ex(nb=64), -3), (ex(h=fake + 2), -1)]:
        assert rc == want
    assert lib.ds_linear_ce_eval_workspace_bytes(2, 0, 64, 16, 64) == 0
    assert lib.ds_bin_expect_eval_workspace_bytes(9, 8, 64, 16, 64) == 0
    assert lib.ds_bin_expect_fwd(fake, 64, fake, fake, 2, 8, 64, 16, fake, None, fake, big, None) == -1


def test_refusals_on_the_host():
    """CPU tensors, and every wrong argument of the C entries, before any launch."""
    from depth_estimation_amd import _lib as L, metrics, synthesis
    with pytest.raises(RuntimeError, match="GPU"):
        metrics.linear_cross_entropy(torch.zeros(2, 4), torch.zeros(3, 4), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="GPU"):
        synthesis.depth_from_bins(torch.zeros(2, 4), torch.zeros(3, 4), torch.zeros(3))
    with pytest.raises(RuntimeError, match="reduction"):
        metrics.linear_cross_entropy(torch.zeros(2, 4), torch.zeros(3, 4), torch.zeros(2, dtype=torch.int64), reduction="avg")
    if not os.path.exists(L.LIB_PATH):
        pytest.skip("libdepthsynth.so not built (run __graft_entry__.build())")
    lib, fake = L.lib(), 0x1000
    big = 1 << 40

    def fwd(h=fake, ldh=64, w=fake, t=fake, dt=2, n=8, d=64, v=16, red=2, out=fake, saved=fake, ws=fake, nb=big):
        return lib.ds_linear_ce_fwd(h, ldh, w, t, dt, n, d, v, -100, red, out, saved, ws, nb, None)

    def bwd(g=fake, gh=fake, gw=fake, ws=fake, nb=big, w=fake, dt=2, ldh=64):
        return lib.ds_linear_ce_bwd(fake, ldh, w, fake, g, dt, 8, 64, 16, -100, 2, fake, gh, gw, ws, nb, None)

    for rc, want in [(fwd(h=None), -1), (fwd(w=None), -1), (fwd(t=None), -1), (fwd(out=None), -1), (fwd(saved=None), -1),
                     (fwd(n=0), -1), (fwd(d=0), -1), (fwd(v=0), -1), (fwd(n=-5), -1), (fwd(ldh=63), -1), (fwd(red=3), -1),
                     (fwd(red=-1), -1), (fwd(dt=3), -2), (fwd(dt=-1), -2), (fwd(n=(1 << 24) + 1), -2),
                     (fwd(d=(1 << 16) + 8, ldh=1 << 20), -2), (fwd(v=(1 << 22) + 1), -2), (fwd(n=1 << 24, v=1 << 22), -2),
                     (fwd(ws=None), -3), (fwd(nb=64), -3), (fwd(ws=fake + 4), -3), (fwd(w=fake + 2), -1),
                     (bwd(g=None), -1), (bwd(gh=None, gw=None), -1), (bwd(gh=fake + 4), -1), (bwd(gw=fake + 4), -1),
                     (bwd(nb=64), -3), (bwd(dt=7), -2), (bwd(ldh=8), -1), (bwd(w=fake + 2), -1)]:
        assert rc == want
    assert lib.ds_linear_ce_workspace_bytes(2, 0, 64, 16, 64, 0) == 0
    assert lib.ds_linear_ce_workspace_bytes(9, 8, 64, 16, 64, 0) == 0
    assert lib.ds_bin_expect_fwd(fake, 64, fake, None, 2, 8, 64, 16, fake, fake, fake, big, None) == -1
    assert lib.ds_bin_expect_bwd(fake, 64, fake, None, fake, 2, 8, 64, 16, fake, fake, fake, fake, big, None) == -1
    assert lib.ds_bin_expect_fwd(fake + 2, 64, fake, fake, 2, 8, 64, 16, fake, fake, fake, big, None) == -1


@pytest.mark.gpu
def test_refusals_of_tensors():
    from depth_estimation_amd import metrics, synthesis
    h, w = torch.zeros(4, 8, device=DEV), torch.zeros(5, 8, device=DEV)
    t, c = torch.zeros(4, dtype=torch.int64, device=DEV), torch.zeros(5, device=DEV)
    for args in [(h.bfloat16(), w, t), (h.double(), w.double(), t), (h[:, :7], w, t), (h, w[0], t), (h, w, t[:3]),
                 (h, w, t.float()), (h, w, t.bool()), (h, w, t.cpu()), (h, w.cpu(), t), (h, w[:0], t),
                 (h[:, :0], w[:, :0], t)]:
        with pytest.raises(RuntimeError):
            metrics.linear_cross_entropy(*args)
    for args in [(h, w, c[:4]), (h, w, c.double()), (h, w, c.cpu()), (h.half(), w, c), (h, w, c.clone().requires_grad_(True))]:
        with pytest.raises(RuntimeError):
            synthesis.depth_from_bins(*args)
    with pytest.raises(RuntimeError, match="ignore_index"):
        metrics.linear_cross_entropy(h, w, t, ignore_index=2 ** 64 - 100)
    wide = torch.empty(2 ** 32 + 5, 1, dtype=torch.float16, device=DEV)      # as a 32-bit number of classes: five
    with pytest.raises(RuntimeError, match="too large"):
        metrics.linear_cross_entropy(h[:, :1].half(), wide, t)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [16384, 16385, 40000, 131072, 131073, 300000])
def test_many_rows_are_listed_in_order(n):
    """Rows left out here and there: every kept row's loss and gradient comes back to its own place."""
    d, v = 8, 4
    h, w, t, up, _ = _data(n, d, v, torch.float32, seed=n, keep=0.37)
    out, gh, gw, tol, th, tw = _oracle(h, w, t=t, up=up)
    got = _ce(h, w, t, "none", up)
    _close(got[0], out, tol, "loss")
    _close(got[1], gh, th, "g_hidden")
    _close(got[2], gw, tw, "g_weight")
    mean = _ce(h, w, t, "mean")[0].double()
    kept = t != -100
    assert abs(float(mean - out[kept].mean())) <= float(tol[kept].mean()) + 2.0 ** -23 * float(mean)
