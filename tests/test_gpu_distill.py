"""Distillation against float64: divergence, log probability of the targets, their gradient.

Tolerances count roundings.  A logarithm of a probability is (x - M) / T minus a logarithm of a sum: the exponents (x - M) / T are off by three
roundings of 2^-24 of themselves, an exponential by 2^-22 relative, sums by some 2^-20 at most: E = 2^-20 (1 + |ln p|).  A gradient's
terms are off by 2^-20 (2 + |ln p|) of themselves, and the whole is rounded once to its type.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}
IGNORE = -100


def _inputs(rows, classes, k, dtype, seed=0, pad=0, empty=True, spread=2.5):
    torch.manual_seed(seed)
    x = (spread * torch.randn(rows, classes + pad, device=DEV)).to(dtype)[:, :classes]
    best, at = (x.float() + torch.randn(rows, classes, device=DEV)).topk(k, 1)
    z = (1.3 * best).to(dtype)
    if empty and k > 1:
        at = torch.where(torch.rand(rows, k, device=DEV) < 0.2, -1, at)
        at[0] = -1
    targets = torch.randint(0, classes, (rows,), device=DEV)
    targets[-1] = IGNORE
    return x, z, at, targets, torch.rand(rows, device=DEV), -torch.rand(rows, device=DEV)


def _exact(x, z, at, tau, targets, g, gl):
    """Values with what each may be off by."""
    given = at >= 0
    log_t = torch.log_softmax((z.double() / tau).masked_fill(~given, float("-inf")), 1)
    t = torch.where(given, log_t.exp(), 0.0).nan_to_num(0.0)
    xd = x.double()
    log_p, log_p1 = torch.log_softmax(xd / tau, 1), torch.log_softmax(xd, 1)
    at0 = at.clamp(min=0)
    lp = log_p.gather(1, at0)
    terms = torch.where(t > 0, t * (log_t - lp), 0.0)
    size = torch.where(t > 0, t * (2 + log_t.abs() + lp.abs()), 0.0)
    out = dict(divergence=(terms.sum(1), 2.0 ** -20 * size.sum(1)))
    some = (t.sum(1) > 0).double()
    p, p1 = log_p.exp(), log_p1.exp()
    gd = (g.double() * some / tau)[:, None]
    grad = gd * p
    e = 2.0 ** -20 * (gd * p * (2 + log_p.abs())).nan_to_num(0.0)
    grad.scatter_add_(1, at0, -gd * t)
    e.scatter_add_(1, at0, 2.0 ** -20 * gd * (t * (2 + log_t.abs())).nan_to_num(0.0))
    if targets is not None:
        counts = targets != IGNORE
        tg = torch.where(counts, targets, 0)[:, None]
        value = torch.where(counts, log_p1.gather(1, tg)[:, 0], 0.0)
        out["log_prob"] = value, 2.0 ** -20 * (1 + value.abs())
        gld = torch.where(counts, gl.double(), 0.0)[:, None]
        grad = grad - gld * p1
        grad.scatter_add_(1, tg, gld)
        e = e + 2.0 ** -20 * (gld.abs() * p1 * (2 + log_p1.abs())).nan_to_num(0.0)
        e.scatter_add_(1, tg, 2.0 ** -23 * gld.abs())
    out["grad"] = grad, e
    return out


def _near(got, want, name):
    value, error = want
    off = (got.double() - value).abs()
    allowed = error + U[got.dtype] * value.abs() * (1 + 2.0 ** -8) + TINY[got.dtype]
    assert bool((off <= allowed).all()), f"{name}: {off.max():.3e}, worst ratio {(off / allowed).max():.3f}"


def _call(x, z, at, tau, targets, g, gl, leaf=None):
    """Outputs and the gradient with respect to x, a view of `leaf` where that is given."""
    from addernetcuda_b200.distill import distillation
    leaf = x.detach().requires_grad_() if leaf is None else leaf
    r = distillation(leaf, z, at, tau, targets, IGNORE)
    outputs, grads = ([r.divergence], [g]) if targets is None else ([r.divergence, r.log_prob], [g, gl])
    return r, torch.autograd.grad(outputs, leaf, grads)[0]


SIZES = [(1, 1, 1), (3, 2, 2), (5, 10, 4), (64, 1000, 20), (7, 1001, 33), (2, 4097, 64), (1300, 3000, 5), (3, 32000, 32), (30, 50257, 8), (700, 10001, 256),
         (1, 128000, 100), (200, 16384, 1)]


@pytest.mark.parametrize("rows,classes,k", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tau,targeted", [(1.0, False), (1.0, True), (2.5, True), (0.6, False)])
def test_values_and_gradient(rows, classes, k, dtype, tau, targeted):
    x, z, at, targets, g, gl = _inputs(rows, classes, k, dtype, seed=rows + k)
    targets = targets if targeted else None
    r, grad = _call(x, z, at, tau, targets, g, gl)
    want = _exact(x, z, at, tau, targets, g, gl)
    _near(r.divergence, want["divergence"], "divergence")
    if targeted:
        _near(r.log_prob, want["log_prob"], "log_prob")
    else:
        assert r.log_prob is None
    assert grad.dtype == dtype
    _near(grad, want["grad"], "grad")


@pytest.mark.parametrize("pad", [1, 3, 8, 47])
def test_padded_rows_and_other_types(pad):
    x, z, at, targets, g, gl = _inputs(37, 1505, 9, torch.bfloat16, seed=pad, pad=pad)
    r, grad = _call(x, z.float() + 5.0, at.int(), 2.0, targets.int(), g, gl, leaf=x.requires_grad_())
    want = _exact(x.detach(), z.float() + 5.0, at, 2.0, targets, g, gl)
    for name, got in (("divergence", r.divergence), ("log_prob", r.log_prob), ("grad", grad)):
        _near(got, want[name], name)


def test_a_class_named_twice_and_as_the_target():
    x, z, at, targets, g, gl = _inputs(50, 300, 6, torch.float32, seed=3, empty=False)
    at[:, 3] = at[:, 0]
    at[:, 5] = at[:, 0]
    targets[:] = at[:, 0]
    r, grad = _call(x, z, at, 1.7, targets, g, gl)
    want = _exact(x, z, at, 1.7, targets, g, gl)
    _near(r.divergence, want["divergence"], "divergence")
    _near(grad, want["grad"], "grad")


@pytest.mark.parametrize("classes", [40, 3000, 40000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_special_rows(classes, dtype):
    x, z, at, targets, g, gl = _inputs(9, classes, 4, dtype, seed=5, empty=False)
    ninf, inf, nan = float("-inf"), float("inf"), float("nan")
    x[0] = ninf                                   # nothing left
    x[1, classes // 2] = nan
    x[2, 1] = inf
    x[3] = ninf                                   # but for what the teacher names
    x[3].scatter_(0, at[3], torch.tensor([1.0, 2.0, 0.5, 0.0], device=DEV).to(dtype))
    x[4, at[4, 1]] = ninf                         # a class of the teacher's that is out
    z[5] = ninf                                   # no class with a share
    z[6, 2] = nan
    at[7, 0] = classes                            # no class
    targets[3] = at[3, 0]
    targets[8] = classes
    r, grad = _call(x, z, at, 2.0, targets, g, gl)
    d, lp = r.divergence, r.log_prob
    assert d[0] == inf and lp[0] == ninf and (grad[0] == 0).all()
    for i in (1, 2):
        assert d[i].isnan() and lp[i].isnan() and grad[i].isnan().all()
    want = _exact(x[3:5], z[3:5], at[3:5], 2.0, targets[3:5], g[3:5], gl[3:5])
    assert torch.isfinite(d[3]) and d[4] == inf and torch.isfinite(lp[3:5]).all()
    assert abs(d[3].double() - want["divergence"][0][0]) <= want["divergence"][1][0]
    _near(grad[3:5], want["grad"], "grad")
    out = x[3] == ninf
    assert (grad[3][out] == 0).all()
    assert d[5] == 0 and torch.isfinite(grad[5]).all()
    only_labels = _exact(x[5:6], z[5:6], torch.full_like(at[5:6], -1), 2.0, targets[5:6], g[5:6], gl[5:6])
    _near(grad[5:6], only_labels["grad"], "grad")
    assert d[6].isnan() and d[7].isnan() and grad[7].isnan().all() and torch.isfinite(lp[6:8]).all()
    assert lp[8].isnan() and torch.isfinite(d[8]) and grad[8].isnan().all()


@pytest.mark.parametrize("classes", [40, 3000, 40000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_nan_stays(classes, dtype):
    """Beside nothing but -inf, and wherever in the row it stands."""
    places = [0, 1, 7, classes // 2, classes - 2, classes - 1]
    x, z, at, targets, g, gl = _inputs(2 * len(places), classes, 4, dtype, seed=6, empty=False)
    x[::2] = float("-inf")
    for i, place in enumerate(places):
        x[2 * i:2 * i + 2, place] = float("nan")
    r, grad = _call(x, z, at, 2.0, targets, g, gl)
    assert r.divergence.isnan().all() and r.log_prob[:-1].isnan().all() and grad.isnan().all()


def test_far_values():
    """Logits of 1e4 and beyond, and a mask of the type's lowest value."""
    for dtype in (torch.float32, torch.bfloat16):
        x, z, at, targets, g, gl = _inputs(20, 2000, 8, dtype, seed=7, empty=False)
        x = x + 20000
        x[:, ::3] = torch.finfo(dtype).min
        z = x.gather(1, at)
        targets = at[:, 0].clone()
        r, grad = _call(x, z, at, 1.5, targets, g, gl)
        keep = (x.gather(1, at) > 0).all(1)
        want = _exact(x, z, at, 1.5, targets, g, gl)
        # exponents are differences of values held to 2^-24: those of far values are exact, as x is
        _near(r.divergence[keep], (want["divergence"][0][keep], want["divergence"][1][keep]), "divergence")
        _near(grad[keep], (want["grad"][0][keep], want["grad"][1][keep]), "grad")
        assert (grad[:, ::3][keep][targets[keep] % 3 != 0] <= 1e-30).all()


def test_gradient_against_differences():
    x, z, at, targets, g, gl = _inputs(6, 50, 5, torch.float32, seed=8, empty=False)
    _, grad = _call(x, z, at, 2.0, targets, g, gl)

    def f(v):
        log_t = torch.log_softmax(z.double() / 2, 1)
        lp = torch.log_softmax(v / 2, 1).gather(1, at)
        counts = targets != IGNORE
        lt = torch.log_softmax(v, 1).gather(1, torch.where(counts, targets, 0)[:, None])[:, 0]
        return (g.double() * (log_t.exp() * (log_t - lp)).sum(1)).sum() + (gl.double() * lt * counts).sum()

    v = torch.randn(6, 50, device=DEV, dtype=torch.float64)
    slope = (f(x.double() + 1e-5 * v) - f(x.double() - 1e-5 * v)) / 2e-5
    assert abs((grad.double() * v).sum() - slope) <= 1e-5 * (1 + abs(slope))


def test_gradients_of_some_shapes_and_refusals():
    from addernetcuda_b200.distill import DistillationLoss, distillation
    x, z, at, targets, g, gl = _inputs(12, 64, 3, torch.float32, seed=9)
    leaf = x.clone().requires_grad_()
    r = distillation(leaf.view(3, 4, 64), z.view(3, 4, 3), at.view(3, 4, 3), 3.0, targets.view(3, 4))
    assert r.divergence.shape == r.log_prob.shape == (3, 4)
    only_d = torch.autograd.grad(r.divergence, leaf, g.view(3, 4), retain_graph=True)[0]
    only_l = torch.autograd.grad(r.log_prob, leaf, gl.view(3, 4))[0]
    _near(only_d, _exact(x, z, at, 3.0, None, g, gl)["grad"], "divergence alone")
    _near(only_l, _exact(x, z, at, 3.0, targets, torch.zeros_like(g), gl)["grad"], "log_prob alone")
    loss = DistillationLoss(3.0, 0.7)(x, targets, z, at)
    want = _exact(x, z, at, 3.0, targets, g, gl)
    counts = targets != IGNORE
    ref = (0.7 * 9 * want["divergence"][0] * counts - 0.3 * want["log_prob"][0]).sum() / counts.sum()
    assert abs(loss - ref) <= 1e-5 * abs(ref)
    grad, = torch.autograd.grad(distillation(leaf, z, at).divergence.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        grad.sum().backward()
    assert distillation(x[:0], z[:0], at[:0]).divergence.shape == (0,)
    one = distillation(x[0], z[0], at[0])
    assert one.divergence.shape == () and one.divergence == 0
    for bad, kind in ((lambda: distillation(x, z[:5], at), ValueError), (lambda: distillation(x, z, at[:, :2]), ValueError),
                      (lambda: distillation(x, z[:, :0], at[:, :0]), ValueError), (lambda: distillation(x, z, at, temperature=0.0), ValueError),
                      (lambda: distillation(x, z, at, temperature=float("inf")), ValueError), (lambda: distillation(x, z, at.float()), TypeError),
                      (lambda: distillation(x, z, at, targets=targets[:3]), ValueError), (lambda: distillation(x, z.cpu(), at), RuntimeError),
                      (lambda: distillation(x.cpu(), z, at), RuntimeError), (lambda: distillation(x.double(), z, at), TypeError),
                      (lambda: distillation(x, z.clone().requires_grad_(), at), RuntimeError), (lambda: DistillationLoss(alpha=2.0), ValueError)):
        with pytest.raises(kind):
            bad()


def test_captured_and_on_another_stream():
    cases = [_inputs(*size, torch.bfloat16, seed=i) for i, size in enumerate(((3, 40000, 16), (400, 5000, 8), (256, 1000, 20)))]
    run = lambda c: [t.clone() for t in (lambda r, grad: (r.divergence, r.log_prob, grad))(*_call(c[0], c[1], c[2], 2.0, *c[3:]))]
    want = [run(c) for c in cases]
    s = torch.cuda.Stream()
    for c, w in zip(cases, want):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got = run(c)
        s.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, w))
        del got
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = run(c)
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, w))


def test_offsets_beyond_32_bits():
    rows, classes = 17000, 128000
    x = torch.zeros(rows, classes, dtype=torch.bfloat16, device=DEV)
    torch.manual_seed(1)
    x[-2:] = torch.randn(2, classes, device=DEV)
    at = torch.arange(8, device=DEV).expand(rows, 8).contiguous() + classes - 8
    z = torch.randn(rows, 8, device=DEV)
    g, targets = torch.ones(rows, device=DEV), torch.full((rows,), classes - 1, device=DEV)
    r, grad = _call(x, z, at, 2.0, targets, g, -g)
    r2, grad2 = _call(x[-2:].clone(), z[-2:], at[-2:], 2.0, targets[-2:], g[-2:], -g[-2:])
    assert torch.allclose(r.divergence[-2:], r2.divergence, rtol=1e-5) and torch.allclose(r.log_prob[-2:], r2.log_prob, rtol=1e-5)
    assert torch.allclose(grad[-2:].float(), grad2.float(), rtol=2 ** -6, atol=1e-9)


def test_training_step_with_a_teacher():
    """A captured step of a small network with a teacher does what the same steps in elementary operations do."""
    from addernetcuda_b200.distill import DistillationLoss
    from addernetcuda_b200.train import TrainStep

    def net(seed):
        torch.manual_seed(seed)
        return torch.nn.Sequential(torch.nn.Flatten(), torch.nn.Linear(48, 64), torch.nn.ReLU(), torch.nn.Linear(64, 30)).to(DEV)

    teacher, student, plain = net(0), net(1), net(1)
    images, labels = torch.randn(16, 3, 4, 4, device=DEV), torch.randint(0, 30, (16,), device=DEV)
    step = TrainStep(student, (16, 3, 4, 4), 30, lr=0.1, momentum=0.0, criterion=DistillationLoss(2.0, 0.5, top_k=6), teacher=teacher)
    opt = torch.optim.SGD(plain.parameters(), lr=0.1)
    for _ in range(3 + 2):      # three steps before the capture, and the replays
        opt.zero_grad()
        out = plain(images)
        best, at = torch.log_softmax(teacher(images), 1).detach().topk(6, 1)
        log_t = torch.log_softmax(best / 2, 1)
        kl = (log_t.exp() * (log_t - torch.log_softmax(out / 2, 1).gather(1, at))).sum(1).mean()
        loss = 0.5 * 4 * kl + 0.5 * torch.nn.functional.cross_entropy(out, labels)
        loss.backward()
        opt.step()
    step.step(images, labels)
    got = step.step(images, labels)
    assert abs(got - loss) <= 1e-4 * abs(loss)
    for a, b in zip(student.parameters(), plain.parameters()):
        assert torch.allclose(a, b, rtol=1e-3, atol=1e-5)
    default = TrainStep(net(2), (16, 3, 4, 4), 30, use_graph=False, teacher=teacher)
    assert torch.isfinite(default.step(images, labels))
