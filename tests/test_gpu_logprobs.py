"""Log probabilities, entropy, top classes and their gradient against float64.

Tolerances count roundings.  The sum of exponentials s >= 1 has terms e^(x - M) of at most three roundings and the error of the exponential
(2^-22, and 2^-24 times its argument, whose weight x e^x is below 0.53) and is added up in at most V / 512 + 16 steps a thread, so ln s
and what is made of it are within K 2^-24 of their scale, K = 64 + V / 256.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _logits(rows, v, dtype, seed=0, spread=2.5):
    torch.manual_seed(seed)
    return (torch.randn(rows, v) * spread).to(dtype).to(DEV), torch.randint(0, v, (rows,), device=DEV)


def _best(x, k):
    """Indices of the k largest, ties to the lowest index."""
    return torch.sort(x.float() + 0.0, dim=1, descending=True, stable=True).indices[:, :k]


def _exact(x, t, k, ignore=-100):
    xd = x.double()
    d = xd - xd.amax(1, keepdim=True)      # the maximum first: even 64 bits lose ln V beside 3e38
    logp = d - d.exp().sum(1, keepdim=True).log()
    p = logp.exp()
    out = {"logp": logp, "p": p, "entropy": -torch.where(p > 0, p * logp, 0.0).sum(1)}
    given = t != ignore
    out["log_prob"] = torch.where(given, logp.gather(1, torch.where(given, t, 0)[:, None])[:, 0], 0.0)
    if k:
        out["idx"] = _best(x, k)
        out["top"] = logp.gather(1, out["idx"])
    return out


def _close(name, got, want, limit):
    assert got.shape == want.shape, name
    same = (got == want.to(got.dtype)) | (got.isnan() & want.isnan())
    off = torch.where(same, 0.0, (got.double() - want).abs())
    limit = torch.where(same, 1.0, limit)
    assert bool((off <= limit).all()), f"{name}: off by {float(off.max()):.3e}, {float((off / limit).max()):.2f} of what is allowed"


def _k(v):
    return (64 + v / 256) * 2.0 ** -24


def _check(x, t, k=0, entropy=True, grads=True, ignore=-100, e=None):
    from addernetcuda_b200.logprobs import token_log_probs
    v = x.shape[-1]
    leaf = x.detach().requires_grad_(grads)
    r = token_log_probs(leaf, t, top_k=k, entropy=entropy, ignore_index=ignore)
    want = _exact(x, t, k, ignore)
    e = e or _k(v)
    _close("log_prob", r.log_prob, want["log_prob"], e * (1 + want["log_prob"].abs()))
    if entropy:
        _close("entropy", r.entropy, want["entropy"], 2 * e * (1 + want["entropy"]))
    if k:
        assert torch.equal(r.top_indices, want["idx"]), (r.top_indices - want["idx"]).nonzero()[:4]
        _close("top", r.top_log_probs, want["top"], e * (1 + want["top"].abs()))
    if not grads:
        return r
    g, ge = torch.randn_like(r.log_prob), torch.randn_like(r.log_prob) if entropy else None
    gt = torch.randn_like(r.top_log_probs) if k else None
    outs, ups = [r.log_prob], [g]
    if entropy:
        outs.append(r.entropy); ups.append(ge)
    if k:
        outs.append(r.top_log_probs); ups.append(gt)
    dx, = torch.autograd.grad(outs, leaf, ups)
    assert dx.dtype == x.dtype and dx.shape == x.shape
    given = t != ignore
    up = torch.zeros_like(x, dtype=torch.float64)
    rows = torch.arange(x.shape[0], device=x.device)
    up[rows[given], t[given]] = g[given].double()
    if k:
        up.scatter_add_(1, want["idx"], gt.double())
    size = up.abs().sum(1, keepdim=True) * want["p"] + up.abs()
    total = up - want["p"] * up.sum(1, keepdim=True)
    if entropy:
        lp = torch.where(want["p"] > 0, want["logp"], 0.0)
        part = -ge.double()[:, None] * want["p"] * (lp + want["entropy"][:, None])
        total = total + part
        size = size + ge.double().abs()[:, None] * want["p"] * (lp.abs() + want["entropy"][:, None] + 1)
    _close("grad", dx, total, U[x.dtype] * total.abs() + TINY[x.dtype] + 2 * e * size + 1e-37)
    return r


SIZES = [1, 2, 3, 7, 8, 10, 31, 33, 100, 127, 255, 257, 1000, 1001, 1023, 1024, 1025, 1031, 2048, 4097, 8191, 8192, 8193, 16385, 32000, 50257, 65537,
         131073]


@pytest.mark.parametrize("v", SIZES)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_every_output_and_gradient(v, dtype):
    for rows, k in ((3, 0), (5, min(v, 5)), (2, min(v, 32))):
        x, t = _logits(rows, v, dtype, seed=v + k)
        _check(x, t, k)


@pytest.mark.parametrize("rows", [1, 2, 4, 18, 37, 74, 148, 149, 300, 1025])
def test_rows_split_over_a_cluster_or_not(rows):
    for v in (1024, 12000, 40001):
        x, t = _logits(rows, v, torch.bfloat16, seed=rows)
        _check(x, t, 20)
        _check(x, t, 1, entropy=False)


@pytest.mark.parametrize("v", [1000, 1025, 4000, 8191, 8192, 8193])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_many_rows(v, dtype):
    """Rows that one warp takes each: a lane adds up V / 32 values, so K = 64 + V / 32."""
    e = (64 + v / 32) * 2.0 ** -24
    for rows, k in ((3551, 5), (3552, 0), (4001, 20)):
        x, t = _logits(rows, v, dtype, seed=v + k)
        t[1::7] = -100
        _check(x, t, k, entropy=k != 0, e=e)


@pytest.mark.parametrize("rows,v", [(2148, 1000003), (600000, 4000)])
def test_offsets_beyond_32_bits(rows, v):
    """The last rows of more than 2^31 logits."""
    from addernetcuda_b200.logprobs import token_log_probs
    assert rows * v > 2 ** 31
    x = torch.zeros(rows, v, dtype=torch.bfloat16, device=DEV)
    tail, t_tail = _logits(8, v, torch.bfloat16, seed=1)
    x[-8:] = tail
    t = torch.zeros(rows, dtype=torch.int64, device=DEV)
    t[-8:] = t_tail
    r = token_log_probs(x.requires_grad_(), t, top_k=3, entropy=True)
    dx, = torch.autograd.grad([r.log_prob, r.entropy], x, [torch.ones_like(r.log_prob), torch.ones_like(r.entropy)])
    tail.requires_grad_()
    w = token_log_probs(tail, t_tail, top_k=3, entropy=True)
    want, = torch.autograd.grad([w.log_prob, w.entropy], tail, [torch.ones_like(w.log_prob), torch.ones_like(w.entropy)])
    e = (64 + v / 32) * 2.0 ** -24      # either variant, each within this of the exact value
    assert torch.equal(r.top_indices[-8:], w.top_indices)
    assert bool(((r.log_prob[-8:] - w.log_prob).abs() <= 2 * e * (1 + w.log_prob.abs())).all())
    assert bool(((r.entropy[-8:] - w.entropy).abs() <= 4 * e * (1 + w.entropy)).all())
    p = torch.log_softmax(tail.detach().double(), 1)
    size = (torch.arange(v, device=DEV) == t_tail[:, None]) + p.exp() * (2 + p.abs() + w.entropy[:, None].double())
    assert bool(((dx[-8:].double() - want.double()).abs() <= 2 * U[torch.bfloat16] * want.double().abs() + 4 * e * size).all())
    assert bool((dx[rows // 2] == dx[0]).all())      # alike rows


@pytest.mark.parametrize("v", [10, 1000, 5000, 50257])
def test_ties_go_to_the_lowest_index(v):
    """Few different values, constant rows, zeros of both signs, runs and strides that meet one thread's share."""
    torch.manual_seed(v)
    x = torch.randint(0, 3, (12, v), device=DEV).float()
    x[1] = 0.5
    x[2] = torch.where(torch.rand(v, device=DEV) < 0.5, 0.0, -0.0)
    x[3] = torch.arange(v, device=DEV) * 1e-3
    x[4] = -x[3]
    x[5] = (torch.arange(v, device=DEV) % 8 == 3).float()
    x[6] = (torch.arange(v, device=DEV) % 4096 < 8).float()
    x[7] = ((torch.arange(v, device=DEV) // 8) % 512 == 5).float() * torch.rand(v, device=DEV)
    x[8] = float("-inf")
    x[8, v // 2:] = 1.0
    x[9] = float("-inf")
    x[9, v // 3] = 2.0
    x[9, v // 2] = 2.0
    t = x.argmax(1)
    for dtype in TYPES:
        for k in (1, 5, min(v, 32)):
            r = _check(x.to(dtype), t, k, grads=False)
            assert bool((r.top_log_probs[:, :1] >= r.top_log_probs).all())


def test_masks_infinities_and_nan():
    from addernetcuda_b200.logprobs import token_log_probs
    inf = float("inf")
    for v in (9, 1000, 6000, 50257, 70001):
        for dtype in TYPES:
            x, t = _logits(9, v, dtype, seed=v)
            low = torch.finfo(dtype).min
            x[0] = torch.where(torch.rand(v, device=DEV) < 0.7, -inf, x[0]); x[0, t[0]] = 1.0
            x[1] = torch.where(torch.rand(v, device=DEV) < 0.7, low, x[1]); x[1, t[1]] = 1.0
            x[2] = low                     # masked with the lowest number throughout: all equal
            x[3] = -inf; x[3, t[3]] = low  # one class left, whatever its logit
            _check(x[:4], t[:4], min(v, 7))
            x[4] = -inf                    # nothing left
            x[5, v // 2] = float("nan")
            x[6, v - 1] = inf
            x[7, 0] = float("nan"); x[7, 1:] = -inf
            leaf = x.detach().requires_grad_()
            r = token_log_probs(leaf, t, top_k=min(v, 7), entropy=True)
            k = r.top_indices.shape[1]
            assert float(r.log_prob[4]) == -inf and float(r.entropy[4]) == 0.0 and bool((r.top_log_probs[4] == -inf).all())
            assert torch.equal(r.top_indices[4], torch.arange(k, device=DEV))
            for i in (5, 6, 7):
                assert bool(r.log_prob[i].isnan()) and bool(r.entropy[i].isnan()) and bool(r.top_log_probs[i].isnan().all())
                assert bool((r.top_indices[i] == -1).all())
            dx, = torch.autograd.grad([r.log_prob, r.entropy, r.top_log_probs], leaf,
                                      [torch.ones_like(r.log_prob), torch.ones_like(r.entropy), torch.ones_like(r.top_log_probs)])
            assert bool((dx[4] == 0).all()) and bool(dx[5:8].isnan().all()) and bool(dx[[0, 1, 2, 3, 8]].isfinite().all())
            r = token_log_probs(leaf, t, entropy=True)
            dx, = torch.autograd.grad(r.log_prob.sum() + r.entropy.sum(), leaf)
            assert bool((dx[0][x[0] == -inf] == 0).all())      # a class that is out gets nothing


def test_large_logits_of_fp32():
    big = 3.0e38
    x = torch.tensor([[big, -big, big], [-big, -big, -big], [1e30, -1e30, 0.0], [-1e38, -1.0000001e38, -3e38]], device=DEV)
    _check(x, torch.tensor([0, 1, 0, 0], device=DEV), 3, grads=False)


def test_ignored_and_impossible_targets():
    from addernetcuda_b200.logprobs import TokenCrossEntropy, token_log_probs
    for v in (50, 3000, 20001):
        x, t = _logits(8, v, torch.float32)
        t[1], t[5] = -100, -100
        r = _check(x, t, 4)
        assert float(r.log_prob[1]) == 0.0
        other = t.clamp(min=0)
        other[2] = 7
        _check(x, other, 4, ignore=7)
        bad = t.clone()
        bad[0], bad[3], bad[4] = v, -1, 1 << 40
        leaf = x.detach().requires_grad_()
        r = token_log_probs(leaf, bad)
        assert r.entropy is None and r.top_indices is None
        dx, = torch.autograd.grad(r.log_prob, leaf, torch.ones_like(r.log_prob))
        for i in range(8):
            wrong = i in (0, 3, 4)
            assert bool(r.log_prob[i].isnan()) == wrong and bool(dx[i].isnan().all() if wrong else dx[i].isfinite().all())
        for reduction in ("mean", "sum", "none"):
            leaf2 = x.detach().requires_grad_()
            loss = TokenCrossEntropy(reduction=reduction)(leaf2, t)
            ref = torch.nn.functional.cross_entropy(x.double(), t, reduction=reduction, ignore_index=-100)
            assert bool(((loss.double() - ref).abs() <= 4 * _k(v) * (8 + ref.abs())).all())      # up to eight terms
            loss.sum().backward()
            xd = x.double().requires_grad_()
            torch.nn.functional.cross_entropy(xd, t, reduction=reduction, ignore_index=-100).sum().backward()
            assert bool(((leaf2.grad.double() - xd.grad).abs() <= 4 * _k(v)).all())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_views_strides_and_alignment(dtype):
    from addernetcuda_b200.logprobs import token_log_probs
    for v in (999, 1000, 10000, 10007):
        buf = torch.randn(6, v + 24, device=DEV).to(dtype) * 2
        for x in (buf[:, :v], buf[:, 8:8 + v], buf[:, 1:1 + v], buf[::2, 5:5 + v], buf[:1, :v].expand(4, v), buf[:, :v].t().contiguous().t()):
            t = torch.randint(0, v, (x.shape[0],), device=DEV)
            _check(x, t, 3)
    x = torch.randn(2, 3, 130, device=DEV).to(dtype)
    t = torch.randint(0, 130, (2, 3), device=DEV)
    a, b = token_log_probs(x[..., :100], t.clamp(max=99), top_k=2), token_log_probs(x[..., :100].reshape(6, 100), t.clamp(max=99).reshape(6), top_k=2)
    assert a.log_prob.shape == (2, 3) and a.top_indices.shape == (2, 3, 2)
    assert torch.equal(a.log_prob.reshape(-1), b.log_prob) and torch.equal(a.top_indices.reshape(6, 2), b.top_indices)
    one = token_log_probs(x[0, 0], t[0, 0], top_k=1)
    assert one.log_prob.shape == () and one.top_indices.shape == (1,)
    assert torch.equal(token_log_probs(x, t.int()).log_prob, token_log_probs(x, t).log_prob)
    assert token_log_probs(x[:0], t[:0], entropy=True).entropy.shape == (0, 3)
    only = token_log_probs(x, entropy=True)
    assert only.log_prob is None and only.top_indices is None


def test_one_output_at_a_time_and_gradients_that_are_views():
    from addernetcuda_b200.logprobs import token_log_probs
    for v in (300, 9000):
        x, t = _logits(4, v, torch.float32)
        want = _exact(x, t, 3)
        for name in ("log_prob", "entropy", "top_log_probs"):
            leaf = x.detach().requires_grad_()
            r = token_log_probs(leaf, t, top_k=3, entropy=True)
            getattr(r, name).sum().backward()       # an expanded gradient
            xd = x.double().requires_grad_()
            logp = torch.log_softmax(xd, 1)
            {"log_prob": logp.gather(1, t[:, None]), "entropy": -(logp.exp() * logp), "top_log_probs": logp.gather(1, want["idx"])}[name].sum().backward()
            assert bool(((leaf.grad.double() - xd.grad).abs() <= 8 * _k(v) * (1 + xd.grad.abs())).all()), name


def test_gradient_against_differences():
    from addernetcuda_b200.logprobs import token_log_probs
    torch.manual_seed(2)
    x, t = torch.randn(2, 9), torch.tensor([3, 8])
    leaf = x.to(DEV).requires_grad_()
    r = token_log_probs(leaf, t.to(DEV), top_k=2, entropy=True)
    (2 * r.log_prob.sum() + 3 * r.entropy.sum() + r.top_log_probs.sum()).backward()
    idx = r.top_indices.cpu()

    def f(v):
        lp = torch.log_softmax(v, 1)
        return 2 * lp.gather(1, t[:, None]).sum() - 3 * (lp.exp() * lp).sum() + lp.gather(1, idx).sum()

    for i in range(2):
        for j in range(9):
            v = x.double()
            v[i, j] += 1e-5
            up = f(v)
            v[i, j] -= 2e-5
            assert abs(float(leaf.grad[i, j]) - float((up - f(v)) / 2e-5)) < 1e-5      # terms of size 10, some 16 fp32 roundings


def test_refusals():
    from addernetcuda_b200.logprobs import token_log_probs
    x, t = _logits(4, 40, torch.float32)
    with pytest.raises(ValueError, match="top_k"):
        token_log_probs(x, t, top_k=33)
    with pytest.raises(ValueError, match="top_k"):
        token_log_probs(x, t, top_k=-1)
    with pytest.raises(ValueError, match="top_k"):
        token_log_probs(x[:, :3], t.clamp(max=2), top_k=4)
    with pytest.raises(ValueError, match="targets have shape"):
        token_log_probs(x, t[:3])
    with pytest.raises(TypeError, match="int64 or int32"):
        token_log_probs(x, t.float())
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        token_log_probs(x.double(), t)
    with pytest.raises(RuntimeError, match="different devices"):
        token_log_probs(x, t.cpu())
    with pytest.raises(ValueError, match="nothing is asked for"):
        token_log_probs(x)
    with pytest.raises(ValueError, match="last axis"):
        token_log_probs(x[:, :0], t)
    leaf = x.requires_grad_()
    g, = torch.autograd.grad(token_log_probs(leaf, t).log_prob.square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_without_the_host_path_the_results_are_the_same(monkeypatch):
    from addernetcuda_b200 import _native
    from addernetcuda_b200.logprobs import token_log_probs

    def run(x, t):
        leaf = x.detach().requires_grad_()
        r = token_log_probs(leaf, t, top_k=4, entropy=True)
        return [*r, torch.autograd.grad(r.log_prob.sum() + r.entropy.sum() + r.top_log_probs.sum(), leaf)[0]]

    for v in (40, 1001, 50257):
        x, t = _logits(3, v, torch.bfloat16)
        a = run(x, t)
        with monkeypatch.context() as m:
            m.setattr(_native, "log_probs", _native._absent)
            b = run(x, t)
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_streams_and_captured_replays():
    from addernetcuda_b200.logprobs import token_log_probs

    def run(x, t):
        leaf = x.detach().requires_grad_()
        r = token_log_probs(leaf, t, top_k=4, entropy=True)
        return [*r, *torch.autograd.grad([r.log_prob, r.entropy], leaf, [torch.ones_like(r.log_prob), torch.ones_like(r.entropy)])]

    for rows, v in ((3, 20000), (400, 5000), (100, 333)):
        x, t = _logits(rows, v, torch.bfloat16)
        want = run(x, t)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = run(x, t)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got))
        xs, ts = x.clone(), t.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run(xs, ts)
        xs.copy_(x.flip(0)); ts.copy_(t.flip(0))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(run(xs, ts), out))


@pytest.mark.parametrize("host_path", [True, False])
def test_gradients_are_not_taken_for_constants(host_path, monkeypatch):
    """A gradient of create_graph=True raises where it is differentiated, beside another term of the loss and for some inputs alone."""
    from addernetcuda_b200 import _native
    from addernetcuda_b200.logprobs import token_log_probs
    if not host_path:
        monkeypatch.setattr(_native, "log_probs", _native._absent)
    x, t = _logits(6, 40, torch.float32)
    for weights in (torch.ones(6, device=DEV), torch.ones(6, device=DEV, requires_grad=True)):
        for part in ("log_prob", "entropy", "top_log_probs"):
            leaf = x.detach().requires_grad_()
            out = getattr(token_log_probs(leaf, t, top_k=3, entropy=True), part)
            total = (out * weights.view([6] + [1] * (out.dim() - 1))).sum()
            g, = torch.autograd.grad(total, leaf, create_graph=True)
            again = getattr(token_log_probs(leaf, t, top_k=3, entropy=True), part)
            assert torch.equal(g.detach(), torch.autograd.grad(again.sum(), leaf)[0])
            with pytest.raises(RuntimeError, match="differentiable once"):
                (total + g.square().sum()).backward(retain_graph=True)
            with pytest.raises(RuntimeError, match="differentiable once"):
                torch.autograd.grad(total + g.square().sum(), leaf, retain_graph=True)
            if weights.requires_grad:
                with pytest.raises(RuntimeError, match="differentiable once"):
                    torch.autograd.grad(g.square().sum(), weights)

def _altered(number, change):
    """Saved-tensor hooks that hand back `change` of the tensor that is saved as the `number`-th."""
    saved = []

    def pack(t):
        saved.append(t)
        return len(saved) - 1, t
    return torch.autograd.graph.saved_tensors_hooks(pack, lambda kept: change(kept[1]) if kept[0] == number else kept[1])


ALTERED = [lambda t: t.to(torch.float16 if t.is_floating_point() else torch.int32), lambda t: t.reshape(-1)[:-1], lambda t: t.cpu()]


@pytest.mark.parametrize("host_path", [True, False])
def test_saved_tensors_that_come_back_in_another_form_are_refused(host_path, monkeypatch):
    from addernetcuda_b200 import _native
    from addernetcuda_b200.logprobs import token_log_probs
    if not host_path:
        monkeypatch.setattr(_native, "log_probs", _native._absent)
    x, t = _logits(6, 40, torch.float32)

    def run(hooks):
        leaf = x.detach().requires_grad_()
        with hooks:
            r = token_log_probs(leaf, t, top_k=3, entropy=True)
        return torch.autograd.grad(r.log_prob.sum() + r.entropy.sum() + r.top_log_probs.sum(), leaf)[0]

    want = run(_altered(-1, None))
    for number in range(5):
        assert torch.equal(run(_altered(number, lambda s: s.clone())), want)
        for change in ALTERED:
            with pytest.raises(RuntimeError, match="saved tensors"):
                run(_altered(number, change))


@pytest.mark.parametrize("host_path", [True, False])
def test_lazily_negated_tensors(host_path, monkeypatch):
    """The imaginary part of a conjugate is one; with one row its strides do not tell."""
    from addernetcuda_b200 import _native
    from addernetcuda_b200.logprobs import token_log_probs
    if not host_path:
        monkeypatch.setattr(_native, "log_probs", _native._absent)
    for rows in (1, 3):
        x, t = _logits(rows, 40, torch.float32)
        leaf = x.detach().requires_grad_()
        negated = lambda v: torch.complex(torch.zeros_like(v), v).conj().imag      # noqa: E731
        up = [torch.rand(rows, device=DEV), torch.rand(rows, device=DEV), torch.rand(rows, 1, device=DEV)]

        def gradient(upstream):
            r = token_log_probs(leaf, t, top_k=1, entropy=True)
            return torch.autograd.grad([r.log_prob, r.entropy, r.top_log_probs], leaf, upstream)[0]

        got, want = gradient([negated(u) for u in up]), gradient([-u for u in up])
        assert torch.equal(got, want)
        assert torch.equal(token_log_probs(negated(x), t).log_prob, token_log_probs(-x, t).log_prob)
