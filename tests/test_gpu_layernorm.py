"""Layer norm (with the sum of a residual stream) against float64: outputs, statistics of what is stored, all gradients.

Tolerances count roundings.  An output of type T is rounded once: half a step, u_T |value| with u = eps / 2.  Before that come fp32
operations; sums are trees or up to D / 32 terms in sequence, whose rounding errors add up like a walk of sqrt(D / 32) steps, so
K = 64 + 4 sqrt(D) roundings of 2^-24 relative to the largest terms that meet in the value are allowed (4: a factor for luck).
"""
import itertools
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}      # half a step of fp16's subnormal numbers


def _inputs(rows, shape, dtype, wtype, residual, seed=0, mean=0.3):
    torch.manual_seed(seed)
    full = (rows, *shape)
    x = (torch.randn(full) * 1.5 + mean).to(dtype).to(DEV)
    r = torch.randn(full).to(dtype).to(DEV) if residual else None
    w = (1 + 0.2 * torch.randn(shape)).to(wtype).to(DEV)
    b = (0.2 * torch.randn(shape)).to(wtype).to(DEV)
    dy, dh = torch.randn(full).to(dtype).to(DEV), torch.randn(full).to(dtype).to(DEV)
    return x, r, w, b, dy, dh


def _exact(x, r, w, b, dy, dh, eps):
    """float64: y, h, dh_total, dw, db, and the scale that the roundings of each are relative to."""
    rows = x.shape[0]
    h = x if r is None else (x.double() + r.double()).to(x.dtype)
    d = h.numel() // max(rows, 1)
    hd = h.double().reshape(rows, d)
    wd = w.double().reshape(d) if w is not None else torch.ones(d, dtype=torch.float64, device=x.device)
    bd = b.double().reshape(d) if b is not None else torch.zeros(d, dtype=torch.float64, device=x.device)
    mu = hd.mean(1, keepdim=True)
    rs = 1 / ((hd - mu).square().mean(1, keepdim=True) + eps).sqrt()
    xh = (hd - mu) * rs
    y = xh * wd + bd
    k = (64 + 4 * math.sqrt(d)) * 2.0 ** -24
    e_xh = k * (hd.abs().amax(1, keepdim=True) * rs + xh.abs())          # error of a normalised value
    out = {"h": h, "y": (y.reshape(x.shape), (e_xh * wd.abs() + k * bd.abs()).reshape(x.shape))}
    if dy is not None:
        dyd = dy.double().reshape(rows, d)
        g = dyd * wd
        m1, m2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
        dx = rs * (g - m1 - xh * m2)
        big = rs * g.abs().amax(1, keepdim=True)
        e_dx = k * big * (2 + xh.abs()) + big * e_xh * (1 + xh.abs())
        if dh is not None:
            dx = dx + dh.double().reshape(rows, d)
            e_dx = e_dx + 2.0 ** -24 * dx.abs()
        kr = (64 + 4 * math.sqrt(rows)) * 2.0 ** -24
        dw, e_dw = (dyd * xh).sum(0), (dyd.abs() * (e_xh + kr * xh.abs())).sum(0)
        db, e_db = dyd.sum(0), kr * dyd.abs().sum(0)
        shape = x.shape[1:]
        out |= {"dx": (dx.reshape(x.shape), e_dx.reshape(x.shape)), "dw": (dw.reshape(shape), e_dw.reshape(shape)),
                "db": (db.reshape(shape), e_db.reshape(shape))}
    return out


def _near(name, got, want, err):
    u, tiny = U[got.dtype], TINY[got.dtype]
    off = (got.double() - want).abs()
    limit = u * (want.abs() + err) + tiny + err
    assert got.shape == want.shape, name
    assert bool((off <= limit).all()), f"{name}: off by {float(off.max()):.3e}, {float((off / limit.clamp(min=1e-300)).max()):.2f} of what is allowed"


def _run(x, r, w, b, dy, dh, eps=1e-5, shape=None):
    from addernetcuda_b200.layernorm import layer_norm
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, r, w, b)]
    out = layer_norm(leaves[0], shape or tuple(x.shape[1:]), leaves[2], leaves[3], eps, residual=leaves[1])
    outs, gs = (list(out), [dy, dh]) if r is not None else ([out], [dy])
    grads = torch.autograd.grad(outs, [t for t in leaves if t is not None], gs)
    return outs, list(grads)


WIDTHS = [1, 2, 3, 8, 31, 33, 64, 127, 128, 250, 256, 257, 511, 512, 520, 1001, 1024, 1032, 2047, 2048, 2056, 4095, 4096, 4104, 8192, 8193,
          8200, 16384, 16392, 16385]


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype,wtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
                                         (torch.float16, torch.float16)], ids=str)
def test_forward_and_gradients(width, dtype, wtype):
    for rows, residual in ((5, False), (3, True)):
        x, r, w, b, dy, dh = _inputs(rows, (width,), dtype, wtype, residual, seed=width + rows)
        outs, grads = _run(x, r, w, b, dy, dh)
        want = _exact(x, r, w, b, dy, dh if residual else None, 1e-5)
        _near("y", outs[0], *want["y"])
        if residual:
            assert torch.equal(outs[1], want["h"])
            assert torch.equal(grads[0], grads[1])
        _near("dx", grads[0], *want["dx"])
        _near("dw", grads[-2], *want["dw"])
        _near("db", grads[-1], *want["db"])


@pytest.mark.parametrize("rows", [1, 2, 7, 148, 297, 1023, 4099])
@pytest.mark.parametrize("width", [24, 384, 1001, 2048])
def test_sums_over_rows(rows, width):
    x, r, w, b, dy, dh = _inputs(rows, (width,), torch.bfloat16, torch.float32, False, seed=rows)
    _, grads = _run(x, r, w, b, dy, dh)
    want = _exact(x, r, w, b, dy, None, 1e-5)
    for name, g in zip(("dx", "dw", "db"), grads):
        _near(name, g, *want[name])
    again = _run(x, r, w, b, dy, dh)[1]
    assert all(torch.equal(a, c) for a, c in zip(grads, again))      # one order of addition


@pytest.mark.parametrize("width", [16400, 32768, 50176, 65544, 131071, 300000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_rows_longer_than_a_block_holds(width, dtype):
    for rows, residual in ((3, True), (64, False)):
        x, r, w, b, dy, dh = _inputs(rows, (width,), dtype, torch.float32, residual, seed=width)
        outs, grads = _run(x, r, w, b, dy, dh)
        want = _exact(x, r, w, b, dy, dh if residual else None, 1e-5)
        _near("y", outs[0], *want["y"])
        _near("dx", grads[0], *want["dx"])
        _near("dw", grads[-2], *want["dw"])
        _near("db", grads[-1], *want["db"])


@pytest.mark.parametrize("rows", [147, 148, 400])
@pytest.mark.parametrize("width", [8200, 12000, 28000, 28672])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_long_rows_enough_for_every_sm(rows, width, dtype):
    """Two rows of one or two arrays in shared memory, or too much for it."""
    for residual in (False, True):
        x, r, w, b, dy, dh = _inputs(rows, (width,), dtype, torch.float32, residual, seed=width)
        outs, grads = _run(x, r, w, b, dy, dh)
        want = _exact(x, r, w, b, dy, dh if residual else None, 1e-5)
        _near("y", outs[0], *want["y"])
        if residual:
            assert torch.equal(outs[1], want["h"])
        _near("dx", grads[0], *want["dx"])
        _near("dw", grads[-2], *want["dw"])
        _near("db", grads[-1], *want["db"])


def test_images_normalised_as_a_whole_and_other_ranks():
    from addernetcuda_b200.layernorm import FusedLayerNorm, layer_norm
    x, _, w, b, dy, _ = _inputs(6, (16, 7, 5), torch.float32, torch.float32, False)
    outs, grads = _run(x, None, w, b, dy, None)
    want = _exact(x, None, w, b, dy, None, 1e-5)
    _near("y", outs[0], *want["y"])
    for name, g in zip(("dx", "dw", "db"), grads):
        _near(name, g, *want[name])
    m = FusedLayerNorm((16, 7, 5)).to(DEV)
    with torch.no_grad():
        m.weight.copy_(w); m.bias.copy_(b)
    assert torch.equal(m(x), outs[0])
    # memory in another order, and leading axes
    assert torch.equal(m(x.to(memory_format=torch.channels_last)), outs[0])
    lead = x.reshape(2, 3, 16, 7, 5)
    assert torch.equal(layer_norm(lead, (16, 7, 5), w, b), outs[0].reshape(lead.shape))
    flat = x.reshape(-1, 5)
    assert layer_norm(flat, 5).shape == flat.shape and layer_norm(flat[0], 5).shape == (5,)
    assert layer_norm(x[:0], (16, 7, 5), w, b).shape == (0, 16, 7, 5)


@pytest.mark.parametrize("given", list(itertools.product([False, True], [False, True])), ids=str)
def test_weight_and_bias_may_be_left_out(given):
    for width in (40, 1001, 20000):
        x, r, w, b, dy, dh = _inputs(4, (width,), torch.float32, torch.float32, True)
        w, b = w if given[0] else None, b if given[1] else None
        outs, grads = _run(x, r, w, b, dy, dh)
        want = _exact(x, r, w, b, dy, dh, 1e-5)
        _near("y", outs[0], *want["y"])
        _near("dx", grads[0], *want["dx"])
        for name, g in zip((["dw"] if given[0] else []) + (["db"] if given[1] else []), grads[2:]):
            _near(name, g, *want[name])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_views_strides_and_alignment(dtype):
    """Rows apart from one another, a base that is not 16-byte aligned, an expanded row, a transposed matrix."""
    from addernetcuda_b200.layernorm import layer_norm
    for width in (64, 1000, 33000):
        buf = torch.randn(5, width + 24, device=DEV).to(dtype)
        w, b = torch.rand(width, device=DEV) + 0.5, torch.randn(width, device=DEV)
        for x in (buf[:, :width], buf[:, 8:8 + width], buf[:, 1:1 + width], buf[::2, 3:3 + width], buf[:1, :width].expand(4, width),
                  buf[:, :width].t().contiguous().t()):
            dense = x.clone(memory_format=torch.contiguous_format)
            xv, xd = x.detach().requires_grad_(), dense.requires_grad_()
            y, yd = layer_norm(xv, width, w, b), layer_norm(xd, width, w, b)
            want = _exact(dense.detach(), None, w, b, torch.ones_like(dense), None, 1e-5)
            _near("y", y, *want["y"])
            _near("y dense", yd, *want["y"])
            g = torch.randn_like(dense)
            a, c = torch.autograd.grad(y, xv, g)[0], torch.autograd.grad(yd, xd, g)[0]
            want = _exact(dense.detach(), None, w, b, g, None, 1e-5)
            _near("dx", a, *want["dx"])
            _near("dx dense", c, *want["dx"])


def test_only_the_gradients_that_are_needed():
    from addernetcuda_b200.layernorm import layer_norm
    x, r, w, b, dy, dh = _inputs(9, (136,), torch.float32, torch.float32, True)
    want = _exact(x, r, w, b, dy, dh, 1e-5)
    names = ("dx", "dx", "dw", "db")
    for i in range(4):
        leaves = [t.detach().requires_grad_(i == j) for j, t in enumerate((x, r, w, b))]
        y, h = layer_norm(leaves[0], 136, leaves[2], leaves[3], residual=leaves[1])
        g = torch.autograd.grad([y, h], leaves[i], [dy, dh]) if i < 2 else torch.autograd.grad(y, leaves[i], dy)
        _near(names[i], g[0], *want[names[i]])
    # only h is used: the norm's part is zero
    xr = x.detach().requires_grad_()
    _, h = layer_norm(xr, 136, w, b, residual=r)
    assert torch.equal(torch.autograd.grad(h, xr, dh)[0], dh)
    # only y
    xr = x.detach().requires_grad_()
    y, _ = layer_norm(xr, 136, w, b, residual=r)
    _near("dx", torch.autograd.grad(y, xr, dy)[0], *_exact(x, r, w, b, dy, None, 1e-5)["dx"])


def test_gradient_against_differences():
    """Central differences of the float64 formula at the kernel's inputs: an independent check of the formulas above."""
    from addernetcuda_b200.layernorm import layer_norm
    torch.manual_seed(1)
    x, w, b, dy = torch.randn(2, 12), torch.rand(12) + 0.5, torch.randn(12), torch.randn(2, 12)
    xg = x.to(DEV).requires_grad_()
    got = torch.autograd.grad(layer_norm(xg, 12, w.to(DEV), b.to(DEV)), xg, dy.to(DEV))[0].double().cpu()

    def loss(v):
        c = v - v.mean(1, keepdim=True)
        return ((c / (c.square().mean(1, keepdim=True) + 1e-5).sqrt() * w.double() + b.double()) * dy.double()).sum()

    e = 1e-5
    for i in range(2):
        for j in range(12):
            v = x.double()
            v[i, j] += e
            up = loss(v)
            v[i, j] -= 2 * e
            assert abs(float(got[i, j]) - float((up - loss(v)) / (2 * e))) < 1e-5 * 10      # fp32 roundings of a dozen terms of size 3


def test_constant_rows_large_means_and_non_finite_rows():
    from addernetcuda_b200.layernorm import layer_norm
    for width in (16, 1001, 2048, 20000):
        w, b = torch.rand(width, device=DEV) + 0.5, torch.randn(width, device=DEV)
        x = torch.full((3, width), 7.25, device=DEV)
        assert torch.equal(layer_norm(x, width, w, b), b.expand(3, width))      # variance 0: 7.25 sums exactly at these widths
        x, _, w, b, dy, _ = _inputs(3, (width,), torch.float32, torch.float32, False, mean=1000.0)
        outs, grads = _run(x, None, w, b, dy, None)
        want = _exact(x, None, w, b, dy, None, 1e-5)
        _near("y", outs[0], *want["y"])
        _near("dx", grads[0], *want["dx"])
        x[1, width // 2] = float("nan")
        x[2, 0] = float("inf")
        y = layer_norm(x, width, w, b)
        assert bool(y[0].isfinite().all()) and bool(y[1].isnan().all()) and bool(y[2].isnan().all())


def test_refusals():
    from addernetcuda_b200.layernorm import layer_norm
    x = torch.randn(4, 8, device=DEV)
    w = torch.ones(8, device=DEV)
    with pytest.raises(ValueError, match="last axes"):
        layer_norm(x, 9)
    with pytest.raises(ValueError, match="last axes"):
        layer_norm(x, (2, 4, 8))
    with pytest.raises(ValueError, match="last axes"):
        layer_norm(x[:, :0], 0)
    with pytest.raises(ValueError, match="weight has shape"):
        layer_norm(x, 8, w[:4])
    with pytest.raises(TypeError, match="weight must be"):
        layer_norm(x, 8, w.half())
    with pytest.raises(TypeError, match="one type"):
        layer_norm(x.bfloat16(), 8, w, w.bfloat16())
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        layer_norm(x.double(), 8)
    with pytest.raises(ValueError, match="residual must have"):
        layer_norm(x, 8, residual=x[:2])
    with pytest.raises(ValueError, match="residual must have"):
        layer_norm(x, 8, residual=x.half())
    with pytest.raises(RuntimeError, match="CUDA"):
        layer_norm(x, 8, w.cpu())
    with pytest.raises(ValueError, match="eps"):
        layer_norm(x, 8, eps=-1.0)
    xr = x.requires_grad_()
    g, = torch.autograd.grad(layer_norm(xr, 8).square().sum(), xr, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_without_the_host_path_the_results_are_the_same(monkeypatch):
    from addernetcuda_b200 import _native
    for width in (24, 1001, 2048, 20000):
        for residual in (False, True):
            args = _inputs(5, (width,), torch.bfloat16, torch.float32, residual)
            outs, grads = _run(*args)
            with monkeypatch.context() as m:
                m.setattr(_native, "layer_norm", _native._absent)
                outs2, grads2 = _run(*args)
            assert all(torch.equal(a, c) for a, c in zip(outs + grads, outs2 + grads2))


def test_streams_and_captured_replays():
    from addernetcuda_b200.layernorm import layer_norm
    x, r, w, b, dy, dh = _inputs(64, (512,), torch.bfloat16, torch.float32, True)
    want = _run(x, r, w, b, dy, dh)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(x, r, w, b, dy, dh)
    side.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(want[0] + want[1], got[0] + got[1]))
    xs, ws = x.clone(), w.clone()
    graphs = []
    for _ in range(2):      # two captured calls, replayed in either order
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _run(xs, r, ws, b, dy, dh)
        graphs.append((g, out))
    for x2, order in ((x, (0, 1)), (x.flip(0).contiguous(), (1, 0))):
        xs.copy_(x2)
        for i in order:
            graphs[i][0].replay()
        torch.cuda.synchronize()
        want = _run(x2, r, w, b, dy, dh)
        for _, out in graphs:
            assert all(torch.equal(a, c) for a, c in zip(want[0] + want[1], out[0] + out[1]))


def test_no_rows():
    from addernetcuda_b200.layernorm import layer_norm
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.randn(0, 33, device=DEV, dtype=dtype, requires_grad=True)
        w, b = (torch.randn(33, device=DEV, requires_grad=True) for _ in range(2))
        y, h = layer_norm(x, 33, w, b, residual=x.detach())
        assert y.shape == h.shape == (0, 33)
        dx, dw, db = torch.autograd.grad(y.sum() + h.sum(), (x, w, b))
        assert dx.shape == (0, 33) and bool((dw == 0).all()) and bool((db == 0).all())


@pytest.mark.parametrize("rows,d", [(530000, 4096), (2150000, 1001)])
def test_offsets_beyond_32_bits(rows, d):
    """The last rows of more than 2^31 elements: rows are summed up alike wherever they lie."""
    from addernetcuda_b200.layernorm import layer_norm
    assert rows * d > 2 ** 31
    tail = torch.randn(8, d, device=DEV, dtype=torch.bfloat16)
    x = torch.zeros(rows, d, device=DEV, dtype=torch.bfloat16)
    x[-8:] = tail
    w, b = (torch.randn(d, device=DEV) for _ in range(2))
    y = layer_norm(x.requires_grad_(), d, w, b)
    hd = tail.double()
    want = (hd - hd.mean(1, keepdim=True)) / (hd.var(1, unbiased=False, keepdim=True) + 1e-5).sqrt()
    k = (64 + 4 * d ** 0.5) * 2.0 ** -24
    top = (want.abs() + 1) * w.double().abs() + b.double().abs()
    off = (y[-8:].double() - (want * w.double() + b.double())).abs()
    assert bool((off <= 2.0 ** -8 * (want * w.double() + b.double()).abs() + 2 * k * top).all())
    dy = torch.zeros_like(x)
    dy[-8:] = torch.randn(8, d, device=DEV)
    dx, = torch.autograd.grad(y, x, dy)
    g = dy[-8:].double() * w.double()
    rstd = 1 / (hd.var(1, unbiased=False, keepdim=True) + 1e-5).sqrt()
    ref = rstd * (g - g.mean(1, keepdim=True) - want * (g * want).mean(1, keepdim=True))
    size = rstd * (g.abs() + g.abs().mean(1, keepdim=True) + (want.abs() + 1) * (g * want).abs().mean(1, keepdim=True))
    assert bool(((dx[-8:].double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 4 * k * size).all())
    assert bool((dx[: 8] == 0).all())


@pytest.mark.parametrize("host_path", [True, False])
@pytest.mark.parametrize("residual", [False, True])
def test_gradients_are_not_taken_for_constants(host_path, residual, monkeypatch):
    """A gradient of create_graph=True that depends on a leaf raises where it is differentiated, beside another term of the loss and for some
    inputs alone; one that depends on nothing is a constant."""
    from addernetcuda_b200 import _native
    from addernetcuda_b200.layernorm import layer_norm
    if not host_path:
        monkeypatch.setattr(_native, "layer_norm", _native._absent)
    x, r, w, b, dy, _ = _inputs(5, (24,), torch.float32, torch.float32, residual)

    def call(leaves, upstream, of):
        """Sum of the outputs weighted by `upstream`, and the gradients of it."""
        out = layer_norm(leaves[0], 24, leaves[2], leaves[3], residual=leaves[1])
        total = (out[0] * upstream).sum() + (out[1] * upstream).sum() if residual else (out * upstream).sum()
        return total, torch.autograd.grad(total, of, create_graph=True)

    for needed in ("x", "r", "w", "all"):
        if needed == "r" and not residual:
            continue
        leaves = [t.clone().requires_grad_(needed in (n, "all")) if t is not None else None for t, n in ((x, "x"), (r, "r"), (w, "w"), (b, "b"))]
        of = [t for t in leaves if t is not None and t.requires_grad]
        for upstream in (dy, dy.clone().requires_grad_()):
            total, grads = call(leaves, upstream, of)
            plain = torch.autograd.grad((lambda o: (o[0] * dy).sum() + (o[1] * dy).sum() if residual else (o * dy).sum())(
                layer_norm(leaves[0], 24, leaves[2], leaves[3], residual=leaves[1])), of)
            assert all(torch.equal(g.detach(), p) for g, p in zip(grads, plain))
            for g, leaf in zip(grads, of):
                const = not upstream.requires_grad and (leaf is leaves[3] or needed == "w")
                if const:
                    assert not g.requires_grad
                    continue
                if leaf is leaves[3]:      # sums of the upstream gradient, the weights of which is its only leaf
                    with pytest.raises(RuntimeError, match="differentiable once"):
                        torch.autograd.grad(g.square().sum(), upstream, retain_graph=True)
                    continue
                with pytest.raises(RuntimeError, match="differentiable once"):
                    (total + g.square().sum()).backward(retain_graph=True)
                with pytest.raises(RuntimeError, match="differentiable once"):
                    torch.autograd.grad(total + g.square().sum(), upstream if upstream.requires_grad else of[0], retain_graph=True)
    only_b = [x, r, w, b.clone().requires_grad_()]
    total, (g,) = call(only_b, dy, [only_b[3]])
    (total + g.square().sum()).backward()
    assert torch.equal(only_b[3].grad, g.detach())


@pytest.mark.parametrize("rows,width", [(3, 16), (3, 33), (3, 600), (3, 1001), (3, 2048), (3, 5000), (3, 20000), (300, 20000), (3, 20001), (3, 70000)])
def test_variances_beyond_the_range_and_of_zero(rows, width):
    """1 / sqrt(infinity) is 0: the norm of such a row is the bias, and no gradient goes through it.  1 / sqrt(0) is infinite."""
    for dtype in (torch.float32, torch.bfloat16):
        x, _, w, b, dy, _ = _inputs(rows, (width,), dtype, dtype, False)
        sign = 1.0 - 2.0 * (torch.arange(width, device=DEV) % 2)
        outs, grads = _run((3e19 * sign).expand(rows, width).to(dtype).contiguous(), None, w, b, dy, None)
        assert torch.equal(outs[0], b.expand(rows, width))
        assert not bool(grads[0].any()) and not bool(grads[1].any())
        outs, _ = _run(x, None, w, b, dy, None, eps=float("inf"))
        assert torch.equal(outs[0], b.expand(rows, width))
        if width % 2 == 0:      # the mean is 0 in any order of addition, the squares are below the smallest number
            outs, _ = _run((1e-30 * sign).expand(rows, width).to(dtype).contiguous(), None, w.abs(), None, dy, None, eps=0.0)
            assert torch.equal(outs[0].float(), (sign * float("inf")).expand(rows, width))

def _altered(number, change):
    """Saved-tensor hooks that hand back `change` of the tensor that is saved as the `number`-th."""
    saved = []

    def pack(t):
        saved.append(t)
        return len(saved) - 1, t
    return torch.autograd.graph.saved_tensors_hooks(pack, lambda kept: change(kept[1]) if kept[0] == number else kept[1])


ALTERED = [lambda t: t.to(torch.float16 if t.is_floating_point() else torch.int32), lambda t: t.reshape(-1)[:-1], lambda t: t.cpu()]


@pytest.mark.parametrize("host_path", [True, False])
@pytest.mark.parametrize("residual", [False, True])
def test_saved_tensors_that_come_back_in_another_form_are_refused(host_path, residual, monkeypatch):
    from addernetcuda_b200 import _native
    from addernetcuda_b200.layernorm import layer_norm
    if not host_path:
        monkeypatch.setattr(_native, "layer_norm", _native._absent)
    x, r, w, b, dy, dh = _inputs(6, (40,), torch.float32, torch.float32, residual)
    _, want = _run(x, r, w, b, dy, dh)
    for number in range(4):
        with _altered(number, lambda t: t.clone()):
            _, got = _run(x, r, w, b, dy, dh)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        for change in ALTERED:
            leaf = x.detach().requires_grad_()
            with _altered(number, change):
                out = layer_norm(leaf, 40, w, b, residual=r)
            with pytest.raises(RuntimeError, match="saved tensors"):
                torch.autograd.grad(out[0] if residual else out, leaf, dy)


def _negated(t):
    """-t, as a lazily negated view of one element or of strided ones."""
    return torch.complex(torch.zeros_like(t), t).conj().imag


@pytest.mark.parametrize("host_path", [True, False])
def test_lazily_negated_tensors(host_path, monkeypatch):
    from addernetcuda_b200 import _native
    from addernetcuda_b200.layernorm import layer_norm
    if not host_path:
        monkeypatch.setattr(_native, "layer_norm", _native._absent)
    x = torch.randn(1, 1, device=DEV)
    assert _negated(x).is_neg() and _negated(x).is_contiguous()
    _, h = layer_norm(_negated(x), 1, residual=_negated(2 * x))
    assert torch.equal(h, -3 * x)
    w, b = torch.full((1,), 2.0, device=DEV), torch.full((1,), 3.0, device=DEV)
    assert float(layer_norm(x, 1, _negated(w), _negated(b))) == -3.0
    for rows, width in ((1, 1), (3, 1), (4, 8)):
        x, _, w, b, dy, _ = _inputs(rows, (width,), torch.float32, torch.float32, False)
        _, want = _run(-x, None, w, b, -dy, None)
        _, got = _run(_negated(x), None, w, b, _negated(dy), None)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
