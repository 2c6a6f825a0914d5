"""RMS norm (with the sum of a residual stream) against float64: outputs, gradients, the output in 8 bits.

Tolerances count roundings.  An output of type T is rounded once: half a step, u_T |value|.  Before that come fp32 operations; sums are
trees or up to D / 32 terms in sequence, so K = 64 + 4 sqrt(D) roundings of 2^-24 relative to the largest terms that meet in the value are
allowed.  A code of 8 bits is off by half a step of e4m3, 2^-4 of its value or 2^-10 (half its subnormal step), times the scale.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}      # half a step of fp16's subnormal numbers
EPS = 1e-6


def _inputs(rows, d, dtype, wtype, residual, seed=0):
    torch.manual_seed(seed)
    x = (torch.randn(rows, d) * 1.5 + 0.3).to(dtype).to(DEV)
    r = torch.randn(rows, d).to(dtype).to(DEV) if residual else None
    w = (1 + 0.2 * torch.randn(d)).to(wtype).to(DEV)
    return x, r, w, torch.randn(rows, d).to(dtype).to(DEV), torch.randn(rows, d).to(dtype).to(DEV)


def _exact(x, r, w, dy, dh, eps=EPS):
    """float64 values and what the fp32 operations may be off by."""
    rows, d = x.shape
    h = x if r is None else (x.double() + r.double()).to(x.dtype)
    hd, wd = h.double(), w.double()
    rs = 1 / (hd.square().mean(1, keepdim=True) + eps).sqrt()
    xh = hd * rs
    k = (64 + 4 * math.sqrt(d)) * 2.0 ** -24
    g = dy.double() * wd
    c = (g * xh).mean(1, keepdim=True)
    dx = rs * (g - xh * c)
    big = (g * xh).abs().mean(1, keepdim=True)
    e_dx = k * rs * (g.abs() + 4 * xh.abs() * big)
    if dh is not None:
        dx = dx + dh.double()
        e_dx = e_dx + 2.0 ** -24 * dx.abs()
    kr = (64 + 4 * math.sqrt(rows)) * 2.0 ** -24
    return dict(h=h, y=(xh * wd, k * (xh * wd).abs()), dx=(dx, e_dx),
                dw=((dy.double() * xh).sum(0), (kr + k) * (dy.double() * xh).abs().sum(0)))


def _near(got, want, name):
    value, error = want
    off = (got.double() - value).abs()
    allowed = error + U[got.dtype] * value.abs() * (1 + 2.0 ** -8) + TINY[got.dtype] + 1e-45
    assert bool((off <= allowed).all()), f"{name}: {off.max():.3e}, allowed there {allowed.flatten()[off.argmax()]:.3e}, worst ratio {(off / allowed).max():.3f}"


SIZES = [(1, 1), (3, 7), (1, 2048), (5, 24), (17, 128), (33, 1000), (300, 513), (7, 1001), (150, 2050), (9, 4096), (4, 8192), (3, 8200), (2, 20001),
         (160, 12000), (2, 70000), (1, 66002)]


@pytest.mark.parametrize("rows,d", SIZES)
@pytest.mark.parametrize("dtype,wtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32)])
@pytest.mark.parametrize("residual", [False, True])
def test_forward_and_gradients(rows, d, dtype, wtype, residual):
    from addernetcuda_b200.rmsnorm import rms_norm
    x, r, w, dy, dh = _inputs(rows, d, dtype, wtype, residual)
    want = _exact(x, r, w, dy, dh if residual else None)
    leaves = [t.requires_grad_() for t in (x, r, w) if t is not None]
    out = rms_norm(x, d, w, EPS, residual=r)
    y, h = out if residual else (out, None)
    _near(y, want["y"], "y")
    if residual:
        assert torch.equal(h, want["h"])
        dx, dr, dw = torch.autograd.grad((y, h), leaves, (dy, dh))
        assert torch.equal(dx, dr)
    else:
        dx, dw = torch.autograd.grad(y, leaves, dy)
    _near(dx, want["dx"], "dx")
    _near(dw, want["dw"], "dw")


@pytest.mark.parametrize("rows,d", SIZES)
@pytest.mark.parametrize("dtype,residual", [(torch.float32, False), (torch.bfloat16, True), (torch.float16, True)])
def test_in_8_bits(rows, d, dtype, residual):
    from addernetcuda_b200.rmsnorm import rms_norm_8bit
    x, r, w, dy, _ = _inputs(rows, d, dtype, dtype, residual, seed=1)
    want = _exact(x, r, w, dy, None)
    out = rms_norm_8bit(x, w, EPS, residual=r)
    if residual:
        out, h = out
        assert torch.equal(h, want["h"])
    value, error = want["y"]
    blocks = -(-d // 128)
    assert out.values.shape == x.shape and out.scales.shape == (rows, blocks) and out.values.stride(0) % 16 == 0
    padded = torch.zeros(rows, blocks * 128, dtype=torch.float64, device=DEV)
    padded[:, :d] = value.abs()
    scale = padded.view(rows, blocks, 128).amax(2) / 448
    k = (68 + 4 * math.sqrt(d)) * 2.0 ** -24
    assert bool(((out.scales.double() - scale).abs() <= k * scale).all())
    each = scale.repeat_interleave(128, 1)[:, :d]
    off = (out.values.double() * out.scales.double().repeat_interleave(128, 1)[:, :d] - value).abs()
    assert bool((off <= (2.0 ** -4 * value.abs() + 2.0 ** -10 * each) * (1 + 4 * k) + error).all())


def test_codes_follow_the_formula():
    """Codes and scales are those of the formula, to the bit, of the norm in 32 bits: rows of fp32 vectors take the same sums with either
    output."""
    from addernetcuda_b200.rmsnorm import rms_norm, rms_norm_8bit
    torch.manual_seed(3)
    for rows, d in ((40, 256), (40, 1024), (3, 1000), (300, 4096), (5, 8192), (200, 60)):
        x = torch.randn(rows, d, device=DEV) * torch.exp(2 * torch.randn(d, device=DEV))
        w = torch.randn(d, device=DEV)
        got, y = rms_norm_8bit(x, w, EPS), rms_norm(x, d, w, EPS)
        blocks = -(-d // 128)
        a = torch.zeros(rows, blocks * 128, device=DEV)
        a[:, :d] = y
        a = a.view(rows, blocks, 128)
        largest = a.abs().amax(2, keepdim=True)
        assert torch.equal(got.scales, (largest * (torch.ones((), device=DEV) / torch.full((), 448.0, device=DEV)))[:, :, 0])
        codes = (a * (largest.reciprocal() * 448)).to(torch.float8_e4m3fn).view(rows, -1)[:, :d]
        assert torch.equal(got.values.float(), codes.float())


def test_special_values():
    from addernetcuda_b200.rmsnorm import rms_norm, rms_norm_8bit
    x = torch.randn(6, 512, device=DEV)
    x[1, 3] = float("nan")
    x[2, 200] = float("inf")
    x[3] = 0
    x[4] = 1e-30
    y = rms_norm(x, 512, None, EPS)
    assert y[1].isnan().all() and y[2, 200].isnan() and (y[2, :200] == 0).all() and (y[3] == 0).all() and torch.isfinite(y[4]).all()
    z = rms_norm_8bit(x, None, EPS)
    v = z.dequantize()
    assert v[1].isnan().all() and v[2, 128:256].isnan().all() and (v[2, :128] == 0).all() and (v[3] == 0).all()
    assert (z.scales[3] == 0).all() and torch.isfinite(v[[0, 3, 4, 5]]).all()
    big = torch.full((1, 256), 3e38, device=DEV)      # squares overflow: 1 / infinity
    assert (rms_norm(big, 256, None, EPS) == 0).all()


def test_views_shapes_and_nothing():
    from addernetcuda_b200.rmsnorm import FusedRMSNorm, rms_norm, rms_norm_8bit
    torch.manual_seed(4)
    whole = torch.randn(5, 7, 300, device=DEV, dtype=torch.bfloat16)
    w = torch.randn(256, device=DEV, dtype=torch.bfloat16)
    for x in (whole[..., 3:259], whole[:, ::2, :256], whole.transpose(0, 1)[..., :256]):
        want = rms_norm(x.contiguous(), 256, w, EPS)
        assert torch.equal(rms_norm(x, 256, w, EPS), want)
        got, ref = rms_norm_8bit(x, w, EPS), rms_norm_8bit(x.contiguous(), w, EPS)
        # another alignment takes another order of the sum: at most a rounding of the scale and a step of some codes
        assert torch.allclose(got.scales, ref.scales, rtol=1e-6) and got.values.shape == x.shape
    assert rms_norm(whole[:0], 300).shape == (0, 7, 300) and rms_norm_8bit(whole[:0]).values.shape == (0, 7, 300)
    x = torch.randn(3, 4, 6, device=DEV, requires_grad=True)
    y = rms_norm(x, (4, 6))
    ref = torch.nn.functional.rms_norm(x.detach().double(), (4, 6), None, 1e-6)
    assert torch.allclose(y.double(), ref, rtol=1e-5, atol=1e-6)
    m, t = FusedRMSNorm(48).to(DEV), torch.nn.RMSNorm(48).to(DEV)
    t.load_state_dict(m.state_dict())
    x = torch.randn(9, 48, device=DEV)
    assert torch.allclose(m(x), t(x), rtol=1e-5, atol=1e-6)
    y, h = m(x, residual=x)
    assert torch.equal(h, x + x) and torch.allclose(y, t(x + x), rtol=1e-5, atol=1e-6)
    with torch.no_grad():
        assert m(x, eight=True).values.dtype == torch.float8_e4m3fn


def test_gradient_against_differences():
    from addernetcuda_b200.rmsnorm import rms_norm
    torch.manual_seed(5)
    x, w, dy = torch.randn(4, 96, device=DEV), torch.randn(96, device=DEV), torch.randn(4, 96, device=DEV, dtype=torch.float64)
    dx, dw = torch.autograd.grad(rms_norm(x.requires_grad_(), 96, w.requires_grad_()), (x, w), dy.float())
    f = lambda a, b: (a / (a.square().mean(1, keepdim=True) + 1e-6).sqrt() * b * dy).sum()
    v, u, step = torch.randn(4, 96, device=DEV, dtype=torch.float64), torch.randn(96, device=DEV, dtype=torch.float64), 1e-5
    xd, wd = x.detach().double(), w.detach().double()
    slope = (f(xd + step * v, wd + step * u) - f(xd - step * v, wd - step * u)) / (2 * step)
    got = (dx.double() * v).sum() + (dw.double() * u).sum()
    assert abs(got - slope) <= 1e-4 * (abs(slope) + 1)


@pytest.mark.parametrize("parts", ["x", "w", "h", "y"])
def test_gradients_of_some(parts):
    from addernetcuda_b200.rmsnorm import rms_norm
    x, r, w, dy, dh = _inputs(40, 264, torch.float32, torch.float32, True, seed=6)
    want = _exact(x, r, w, dy if parts != "h" else torch.zeros_like(dy), dh if parts != "y" else None)
    if parts == "w":
        y, h = rms_norm(x, 264, w.requires_grad_(), EPS, residual=r)
        _near(torch.autograd.grad(y, w, dy)[0], want["dw"], "dw")
        return
    y, h = rms_norm(x.requires_grad_(), 264, w, EPS, residual=r)
    got = torch.autograd.grad(*{"x": ((y, h), x, (dy, dh)), "h": (h, x, dh), "y": (y, x, dy)}[parts])[0]
    _near(got, want["dx"], "dx")


def test_once_differentiable_and_refusals():
    from addernetcuda_b200.rmsnorm import rms_norm, rms_norm_8bit
    x = torch.randn(4, 64, device=DEV, requires_grad=True)
    g, = torch.autograd.grad(rms_norm(x, 64).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.sum().backward()
    with pytest.raises(RuntimeError, match="no gradient"):
        rms_norm_8bit(x)
    x = x.detach()
    for bad, kind in ((lambda: rms_norm(x, 63), ValueError), (lambda: rms_norm(x, 64, torch.ones(64, device=DEV, dtype=torch.bfloat16)), TypeError),
                      (lambda: rms_norm(x.double(), 64), TypeError), (lambda: rms_norm(x, 64, residual=x[:2]), ValueError),
                      (lambda: rms_norm(x, 64, eps=-1.0), ValueError), (lambda: rms_norm(x.cpu(), 64), RuntimeError),
                      (lambda: rms_norm_8bit(x, torch.ones(63, device=DEV)), ValueError), (lambda: rms_norm_8bit(x.cpu()), RuntimeError)):
        with pytest.raises(kind):
            bad()


def test_captured_and_on_another_stream():
    from addernetcuda_b200.rmsnorm import rms_norm, rms_norm_8bit
    x, r, w, dy, dh = _inputs(64, 2048, torch.bfloat16, torch.bfloat16, True, seed=7)
    leaves = [x.requires_grad_(), r.requires_grad_(), w.requires_grad_()]

    def step():
        y, h = rms_norm(x, 2048, w, EPS, residual=r)
        grads = torch.autograd.grad((y, h), leaves, (dy, dh))
        with torch.no_grad():
            z, _ = rms_norm_8bit(x, w, EPS, residual=r)
        return [y, h, *grads, z.values.float(), z.scales]

    want = [t.detach().clone() for t in step()]      # no eager graph of the same leaves lives on
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = step()
    s.synchronize()
    del side
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for t in got:
        t.detach().zero_()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_offsets_beyond_32_bits():
    from addernetcuda_b200.rmsnorm import rms_norm, rms_norm_8bit
    rows, d = 270000, 8200
    x = torch.empty(rows, d, dtype=torch.bfloat16, device=DEV)
    x[-3:] = torch.randn(3, d, device=DEV)
    x[:-3] = 1.0
    with torch.no_grad():
        y = rms_norm(x, d)
        assert torch.equal(y[-3:], rms_norm(x[-3:].clone(), d)) or torch.allclose(y[-3:].float(), rms_norm(x[-3:].clone(), d).float(), rtol=2 ** -7)
        assert bool((y[0] == 1).all())
        del y
        z = rms_norm_8bit(x)
        assert torch.equal(z.values[-3:].float(), rms_norm_8bit(x[-3:].clone()).values.float())
