"""The operators around a head at their edges: modules in place of torch's own, rows that do not count, a teacher that fails, derivatives that
are asked for where there are none."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_the_norm_module_has_torchs_eps(dtype):
    """An eps of None is that of the type that is computed in, float32, on both devices: rows whose mean square is near it show which one was taken."""
    from addernetcuda_b200.rmsnorm import FusedRMSNorm
    torch.manual_seed(0)
    d = 512
    for size in (0.05, 2e-4):
        x, r = ((size * torch.randn(40, d)).to(dtype).to(DEV) for _ in range(2))
        m = FusedRMSNorm(d).to(DEV).to(dtype)
        h = (x.double() + r.double()).to(dtype)
        y, out = m(x, residual=r)
        with torch.no_grad():
            eight = m(x, eight=True).dequantize(torch.float64)
        assert torch.equal(out, h)
        for got, v in ((m(x), x), (y, h)):
            want = v.double() / (v.double().square().mean(-1, keepdim=True) + 2.0 ** -23).sqrt()
            # the sum of squares: d roundings at most of 2^-24 of itself, halved by the root; three more for the root and the products
            allowed = (U[dtype] + (d / 2 + 4) * 2.0 ** -24) * want.abs() * (1 + 2.0 ** -8) + (2.0 ** -25 if dtype == torch.float16 else 0.0)
            assert bool(((got.double() - want).abs() <= allowed).all())
            torchs = torch.nn.RMSNorm(d).to(DEV).to(dtype)(v).double()
            assert bool(((got.double() - torchs).abs() <= 2 * allowed + 2 * U[dtype] * want.abs()).all())
        want = x.double() / (x.double().square().mean(-1, keepdim=True) + 2.0 ** -23).sqrt()
        assert (eight - want).norm() <= 2.0 ** -4 * want.norm()      # half a step of e4m3 each


def _distill_inputs(rows, classes, k, dtype, seed):
    torch.manual_seed(seed)
    x = (2.5 * torch.randn(rows, classes, device=DEV)).to(dtype)
    best, at = (x.float() + torch.randn(rows, classes, device=DEV)).topk(k, 1)
    targets = torch.randint(0, classes, (rows,), device=DEV)
    return x, (1.3 * best).to(dtype), at, targets


@pytest.mark.parametrize("classes", [40, 3000, 40000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_what_the_teacher_says_of_rows_that_do_not_count(classes, dtype):
    """A row that is ignored, and one whose divergence is not asked for, has nothing of the teacher's in its gradient, whatever that is."""
    from addernetcuda_b200.distill import DistillationLoss, distillation
    x, z, at, targets = _distill_inputs(9, classes, 4, dtype, 1)
    targets[:4] = -100
    bad_z, bad_at = z.clone(), at.clone()
    bad_at[0] = -100
    bad_at[1, 2] = classes
    bad_z[2, 1] = float("nan")
    bad_z[3] = float("inf")
    for loss_of in (DistillationLoss(2.0, 0.6), DistillationLoss(1.0, 0.5), DistillationLoss(3.0, 1.0)):
        leaf = x.clone().requires_grad_()
        clean, broken = (loss_of(leaf, targets, *t) for t in ((z, at), (bad_z, bad_at)))
        assert torch.equal(clean, broken) and torch.isfinite(clean)
        want, got = (torch.autograd.grad(t, leaf)[0] for t in (clean, broken))
        assert torch.equal(got, want) and (got[:4] == 0).all() and got[4:].abs().sum() > 0
    leaf = x.clone().requires_grad_()
    want, got = (torch.autograd.grad(distillation(leaf, *t, 2.0, targets.clamp(min=0)).log_prob.sum(), leaf)[0] for t in ((z, at), (bad_z, bad_at)))
    assert torch.equal(got, want) and torch.isfinite(got).all()


@pytest.mark.parametrize("classes", [40, 3000, 40000])
def test_a_teacher_that_fails_is_seen(classes):
    """token_log_probs names no classes in a row with a NaN or an infinity: such a row's divergence is NaN, not that of a row without classes."""
    from addernetcuda_b200.distill import distillation
    from addernetcuda_b200.logprobs import token_log_probs
    x, _, _, targets = _distill_inputs(6, classes, 4, torch.float32, 2)
    teacher = x + torch.randn_like(x)
    teacher[1, 3] = float("nan")
    teacher[4, classes - 1] = float("inf")
    best = token_log_probs(teacher, top_k=4)
    leaf = x.clone().requires_grad_()
    r = distillation(leaf, best.top_log_probs, best.top_indices, 2.0, targets)
    assert r.divergence.isnan().tolist() == [False, True, False, False, True, False] and torch.isfinite(r.log_prob).all()
    grad, = torch.autograd.grad(r.divergence.sum(), leaf)
    assert grad[[1, 4]].isnan().all() and torch.isfinite(grad[[0, 2, 3, 5]]).all()


@pytest.mark.parametrize("use_graph", [False, True])
def test_a_step_with_a_teacher_that_fails(use_graph):
    from addernetcuda_b200.train import TrainStep

    class Teacher(torch.nn.Module):
        def forward(self, images):
            logits = images.flatten(1)[:, :30] * 3
            return torch.where(torch.arange(16, device=DEV)[:, None] == 3, float("nan"), logits)

    torch.manual_seed(3)
    student = torch.nn.Sequential(torch.nn.Flatten(), torch.nn.Linear(48, 30)).to(DEV)
    step = TrainStep(student, (16, 3, 4, 4), 30, teacher=Teacher(), use_graph=use_graph)
    assert step.step(torch.randn(16, 3, 4, 4, device=DEV), torch.randint(0, 30, (16,), device=DEV)).isnan()


def test_a_term_of_weight_0_is_left_out():
    """alpha = 0: an infinite divergence; alpha = 1: a label that the network rules out."""
    from addernetcuda_b200.distill import DistillationLoss
    x, z, at, targets = _distill_inputs(12, 64, 3, torch.float32, 4)
    ruled_out = x.clone()
    ruled_out[0, at[0, 0]] = float("-inf")
    targets[0] = at[0, 1]
    targets[-1] = -100
    counts = targets != -100
    leaf = ruled_out.requires_grad_()
    loss = DistillationLoss(2.0, 0.0)(leaf, targets, z, at)
    want = torch.nn.functional.cross_entropy(leaf.double(), targets)
    assert abs(loss.double() - want) <= 1e-5 * want
    got, ref = torch.autograd.grad(loss, leaf)[0], torch.autograd.grad(want, leaf)[0]
    assert (got.double() - ref).norm() <= 1e-5 * ref.norm()

    out = [c for c in range(64) if c not in at[1].tolist()][0]
    ruled_out = x.clone()
    ruled_out[1, out] = float("-inf")
    targets[1] = out
    leaf = ruled_out.requires_grad_()
    loss = DistillationLoss(2.0, 1.0)(leaf, targets, z, at)
    xd = leaf.double()
    log_t = torch.log_softmax(z.double() / 2, 1)
    each = (log_t.exp() * (log_t - torch.log_softmax(xd / 2, 1).gather(1, at))).sum(1)
    want = 4 * (each * counts).sum() / counts.sum()
    assert abs(loss.double() - want) <= 1e-5 * want
    got, ref = torch.autograd.grad(loss, leaf)[0], torch.autograd.grad(want, leaf)[0]
    assert (got.double() - ref).norm() <= 1e-5 * ref.norm()
    for bad, kind in ((targets[:3], ValueError), (targets.float(), TypeError), (targets.cpu(), RuntimeError)):
        for alpha in (0.0, 0.5, 1.0):
            with pytest.raises(kind):
                DistillationLoss(2.0, alpha)(x, bad, z, at)


def _rows8(m, k, dtype=torch.bfloat16):
    from addernetcuda_b200.rmsnorm import rms_norm_8bit
    with torch.no_grad():
        return rms_norm_8bit(torch.randn(m, k, device=DEV).to(dtype))


def test_a_layer_behind_a_norm_in_8_bits():
    """Linear8bit takes codes, with and without a bias, as linear_8bit does; of several axes; no convolution does."""
    from addernetcuda_b200.linear8 import Linear8bit, Rows8, Weight8, linear_8bit
    torch.manual_seed(5)
    x = _rows8(12, 300)
    for bias in (False, True):
        layer = torch.nn.Linear(300, 70, bias=bias).to(DEV)
        eight = Linear8bit(layer)
        y = eight(x)
        b = layer.bias.detach().bfloat16() if bias else None
        assert y.dtype == torch.bfloat16 and torch.equal(y, linear_8bit(x, Weight8(eight.values, eight.scales), b))
        exact = x.dequantize(torch.float64) @ Weight8(eight.values, eight.scales).dequantize(torch.float64).t() + (b.double() if bias else 0.0)
        assert (y.double() - exact).norm() <= 2.0 ** -8 * exact.norm()
        three = Rows8(x.values.contiguous().view(3, 4, 300), x.scales.view(3, 4, 3))
        assert torch.equal(eight(three), y.view(3, 4, 70))
        assert torch.equal(eight(x, torch.float32), linear_8bit(x, Weight8(eight.values, eight.scales), layer.bias.detach() if bias else None, torch.float32))
    with pytest.raises(TypeError):
        Linear8bit(torch.nn.Conv2d(300, 8, 1).to(DEV))(x)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_layers_bias(dtype):
    """The layer against float64 of its codes, with a bias as large as the product; a layer of its own, whatever becomes of the one it was made of."""
    from addernetcuda_b200.linear8 import Linear8bit, Weight8, quantize_rows
    torch.manual_seed(6)
    for make, x in ((lambda: torch.nn.Linear(200, 130), torch.randn(30, 200, device=DEV)), (lambda: torch.nn.Conv2d(200, 130, 1), torch.randn(2, 200, 3, 5, device=DEV))):
        layer = make().to(DEV)
        with torch.no_grad():
            layer.bias.normal_()
        x = x.to(dtype)
        eight = Linear8bit(layer)
        y = eight(x)
        rows = x if x.dim() == 2 else x.permute(0, 2, 3, 1).reshape(-1, 200)
        exact = quantize_rows(rows).dequantize(torch.float64) @ Weight8(eight.values, eight.scales).dequantize(torch.float64).t() + layer.bias.double().to(dtype).double()
        got = y if x.dim() == 2 else y.permute(0, 2, 3, 1).reshape(-1, 130)
        size = quantize_rows(rows).dequantize(torch.float64).abs() @ Weight8(eight.values, eight.scales).dequantize(torch.float64).abs().t() + layer.bias.double().abs()
        # the output's rounding, 128 + 3 + blocks roundings of 2^-23 of the magnitudes, two of what dequantize rounds
        assert bool(((got.double() - exact).abs() <= U[dtype] * exact.abs() * (1 + 2.0 ** -8) + 140 * 2.0 ** -23 * size).all())
        with torch.no_grad():
            layer.bias.zero_()
            layer.weight.zero_()
        assert torch.equal(eight(x), y)
        state = {k: torch.zeros_like(v.float()).to(v.dtype) for k, v in eight.state_dict().items()}
        with torch.no_grad():
            layer.bias.fill_(1.0)
        eight.load_state_dict(state)
        assert (layer.bias == 1).all() and (eight(x) == 0).all()


def test_a_convolutions_images():
    """What nn.Conv2d takes and gives: an image without a batch, no images, outputs in the order of the input."""
    from addernetcuda_b200.linear8 import Linear8bit
    torch.manual_seed(7)
    conv = torch.nn.Conv2d(40, 24, 1).to(DEV)
    eight = Linear8bit(conv)
    x = torch.randn(3, 40, 5, 7, device=DEV)
    y = eight(x)
    assert y.is_contiguous() and y.view(3, -1).shape == (3, 24 * 35)
    assert torch.equal(eight(x[1]), eight(x[1:2])[0]) and eight(x[1]).is_contiguous()
    last = eight(x.contiguous(memory_format=torch.channels_last))
    assert torch.equal(last, y) and last.is_contiguous(memory_format=torch.channels_last)
    assert eight(x[:0]).shape == conv(x[:0]).shape
    for bad in (x[0, 0], x[None]):
        with pytest.raises(ValueError):
            eight(bad)


def test_which_layers_are_put_in_8_bits():
    """All or none, where one of them cannot be; none whose weight another module reads or computes."""
    import copy
    from torch.nn.utils import prune
    from addernetcuda_b200.inference import quantize_linear
    from addernetcuda_b200.linear8 import Linear8bit
    torch.manual_seed(8)
    for odd, kind in ((torch.nn.Linear(16, 16).to(DEV).double(), TypeError), (torch.nn.Linear(16, 16), RuntimeError)):
        net = torch.nn.Sequential(torch.nn.Linear(16, 16).to(DEV), odd).train()
        with pytest.raises(kind):
            quantize_linear(net)
        assert type(net[0]) is torch.nn.Linear and type(net[1]) is torch.nn.Linear and net.training
    net = torch.nn.Sequential(torch.nn.Linear(32, 64), torch.nn.TransformerEncoder(torch.nn.TransformerEncoderLayer(64, 4, 128, batch_first=True), 2)).to(DEV)
    x = torch.randn(2, 5, 32, device=DEV)
    encoder = copy.deepcopy(net[1]).eval()
    quantize_linear(net)
    assert isinstance(net[0], Linear8bit)
    for no_grad in (False, True):
        with torch.set_grad_enabled(not no_grad):
            assert torch.equal(net(x), encoder(net[0](x)))
    pruned = torch.nn.Linear(16, 16).to(DEV)
    prune.l1_unstructured(pruned, "weight", 0.5)
    net = quantize_linear(torch.nn.Sequential(pruned, torch.nn.Linear(16, 16).to(DEV)))
    assert net[0] is pruned and isinstance(net[1], Linear8bit)
    prune.remove(pruned, "weight")
    assert isinstance(quantize_linear(net)[0], Linear8bit)


def test_derivatives_are_refused():
    """Operators without a gradient raise where one would be recorded, forward-mode tangents and trained scales among them."""
    import torch.autograd.forward_ad as fwd
    from addernetcuda_b200.linear8 import Rows8, Weight8, linear_8bit, quantize_rows, quantize_weight
    from addernetcuda_b200.rmsnorm import rms_norm_8bit
    x, t = torch.randn(4, 128, device=DEV), torch.randn(4, 128, device=DEV)
    w = quantize_weight(torch.randn(64, 128, device=DEV))
    rows = quantize_rows(x)
    b = torch.zeros(64, device=DEV)
    with fwd.dual_level():
        dual = fwd.make_dual(x, t)
        for call in (lambda: quantize_rows(dual), lambda: quantize_weight(dual), lambda: linear_8bit(dual, w), lambda: rms_norm_8bit(dual),
                     lambda: rms_norm_8bit(x, residual=dual), lambda: rms_norm_8bit(x, fwd.make_dual(torch.ones(128, device=DEV), t[0])),
                     lambda: linear_8bit(x, w, fwd.make_dual(b, torch.ones_like(b))),
                     lambda: linear_8bit(Rows8(rows.values, fwd.make_dual(rows.scales, torch.ones_like(rows.scales))), w)):
            for grad in (True, False):      # no_grad is for the backward mode alone
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="no gradient"):
                    call()
        quantize_rows(fwd.unpack_dual(dual).primal)
    for call in (lambda: linear_8bit(Rows8(rows.values, rows.scales.clone().requires_grad_()), w, dtype=torch.float32),
                 lambda: linear_8bit(x, Weight8(w.values, w.scales.clone().requires_grad_()))):
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
        with torch.no_grad():
            assert torch.equal(call(), linear_8bit(x, w))


@pytest.mark.parametrize("rows,classes,k", [(5, 10, 4), (64, 1000, 20), (7, 1001, 33), (1300, 3000, 5), (3, 32000, 32), (30, 50257, 8), (700, 10001, 256), (1, 128000, 100)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tau", [2.0, 4.0])
def test_temperatures_whose_second_exponential_is_a_power(rows, classes, k, dtype, tau):
    from tests.test_gpu_distill import _call, _exact, _inputs, _near
    x, z, at, targets, g, gl = _inputs(rows, classes, k, dtype, seed=rows + k)
    r, grad = _call(x, z, at, tau, targets, g, gl)
    want = _exact(x, z, at, tau, targets, g, gl)
    for name, got in (("divergence", r.divergence), ("log_prob", r.log_prob), ("grad", grad)):
        _near(got, want[name], name)


@pytest.mark.parametrize("classes", [3, 40000])
@pytest.mark.parametrize("dtype,one,least", [(torch.float32, 1.0, 2.0 ** -30), (torch.bfloat16, 1.0, 2.0 ** -30), (torch.float16, 2.0, 2.0 ** -24)])
def test_differences_of_far_probabilities(dtype, one, least, classes):
    """Weights of one and of one - least, in either order, and a border between the two that lies by half of least beside the middle of their sum: it
    shows whether least, which 32 bits cannot hold beside one, is part of the sum."""
    from addernetcuda_b200.drafts import verify_drafts
    p, q = torch.zeros(2, 2, classes, dtype=dtype, device=DEV), torch.zeros(2, 1, classes, dtype=dtype, device=DEV)
    first, second = 0, classes - 2
    p[:, 0, first] = p[:, 0, second] = one
    q[0, 0, second] = least      # weights one, one - least: up to the first it is above the half
    q[1, 0, first] = least       # weights one - least, one: it is below
    q[:, 0, classes - 1] = 0.5   # the drafted class, which the target rules out
    u = torch.tensor([[0.9, 0.5]], device=DEV).expand(2, 2).contiguous()
    r = verify_drafts(p, q, torch.full((2, 1), classes - 1, device=DEV), u)
    assert r.accepted.tolist() == [0, 0] and r.tokens[:, 0].tolist() == [first, second]


@pytest.mark.parametrize("classes", [1001, 4096, 50000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_weights_of_many_sizes(classes, dtype):
    """Probabilities from 1 down to 2^-24, some of which are 0, some negative: as far apart as they come."""
    from addernetcuda_b200.drafts import verify_drafts
    torch.manual_seed(classes)
    b = 60

    def weights(*shape):
        w = torch.exp2(-24 * torch.rand(*shape, device=DEV))
        return torch.where(torch.rand(*shape, device=DEV) < 0.1, 0.0, w).to(dtype)

    p, q = weights(b, 2, classes), weights(b, 1, classes)
    q = torch.where(torch.rand(b, 1, classes, device=DEV) < 0.05, -q, q)
    p[:, 0, 5], q[:, 0, 5] = 0, 1      # the drafted class
    u = torch.rand(b, 2, device=DEV).clamp(min=0.1)
    r = verify_drafts(p, q, torch.full((b, 1), 5, device=DEV), u)
    w = (p[:, 0].double() - q[:, 0].double()).clamp(min=0)      # exact
    reached = w.cumsum(1)
    there = (reached > u[:, 1:].double() * reached[:, -1:]) & (w > 0)
    want = torch.where(there, torch.arange(classes, device=DEV), classes).amin(1)
    assert (r.accepted == 0).all() and torch.equal(r.tokens[:, 0], want)


def test_a_trace_records_the_operators():
    """torch.jit.trace: the traced function follows new inputs, of other lengths too."""
    from addernetcuda_b200.distill import distillation
    from addernetcuda_b200.drafts import verify_drafts
    from addernetcuda_b200.linear8 import Linear8bit, linear_8bit, quantize_rows, quantize_weight
    from addernetcuda_b200.rmsnorm import rms_norm, rms_norm_8bit
    torch.manual_seed(9)
    layer, conv = (Linear8bit(m.to(DEV)) for m in (torch.nn.Linear(100, 70), torch.nn.Conv2d(100, 70, 1)))
    w = quantize_weight(torch.randn(64, 100, device=DEV))
    weight = torch.randn(100, device=DEV)

    def rows(n):
        return (torch.randn(n, 100, device=DEV),)

    def drafts(n):
        p, q = (torch.softmax(torch.randn(n, k, 4000, device=DEV), -1) for k in (3, 2))
        return p, q, torch.randint(0, 4000, (n, 2), device=DEV), torch.rand(n, 3, device=DEV), torch.randint(0, 3, (n,), device=DEV)

    def distilled(n):
        return 2 * torch.randn(n, 100, device=DEV), torch.randn(n, 4, device=DEV), torch.randint(0, 100, (n, 4), device=DEV), torch.randint(0, 100, (n,), device=DEV)

    for call, inputs in ((layer, rows), (conv, lambda n: (torch.randn(n, 100, 2, 3, device=DEV),)), (lambda x: rms_norm(x, 100, weight), rows),
                         (lambda x: tuple(quantize_rows(x)), rows), (lambda x: tuple(quantize_weight(x)), rows), (lambda x: tuple(rms_norm_8bit(x, weight)), rows),
                         (lambda x: linear_8bit(rms_norm_8bit(x, None, 1e-6, x)[0], w), rows), (lambda *a: tuple(verify_drafts(*a)), drafts),
                         (lambda p, q, t, u, n: tuple(verify_drafts(p, None, t.int(), u)), drafts), (lambda x, z, at, t: tuple(distillation(x, z, at, 2.0, t)), distilled)):
        with torch.no_grad():
            traced = torch.jit.trace(call, inputs(3), check_trace=False)
            for n in (3, 5):
                new = inputs(n)
                got, want = traced(*new), call(*new)
                for g, e in zip(*((t,) if isinstance(t, torch.Tensor) else t for t in (got, want))):
                    assert g.dtype == e.dtype and g.shape == e.shape and torch.equal(g.float(), e.float())


def test_a_trace_of_inputs_in_another_order():
    """Rows that have to be copied, within the norms and the losses."""
    from addernetcuda_b200.distill import distillation
    from addernetcuda_b200.layernorm import FusedLayerNorm
    from addernetcuda_b200.logprobs import token_log_probs
    from addernetcuda_b200.rmsnorm import FusedRMSNorm
    torch.manual_seed(10)

    class Of(torch.nn.Module):
        def __init__(self, call):
            super().__init__()
            self.call = call

        def forward(self, x):
            return self.call(x.movedim(-3, -1))

    z, at = torch.randn(2, 4, 5, 3, device=DEV), torch.randint(0, 40, (2, 4, 5, 3), device=DEV)
    for call in (FusedRMSNorm(40), FusedLayerNorm(40), lambda x: token_log_probs(x, at[..., 0]).log_prob, lambda x: distillation(x, z, at).divergence):
        net = Of(call).to(DEV)
        x, new = (torch.randn(2, 40, 4, 5, device=DEV) for _ in range(2))
        for grad in (False, True):
            with torch.set_grad_enabled(grad):
                traced = torch.jit.trace(net, x, check_trace=False)
                assert torch.equal(traced(new), net(new))


def test_a_trace_of_a_network_for_inference():
    """Folded batch norms and a head in 8 bits: the traced network follows new images."""
    from addernetcuda_b200 import resnet
    from addernetcuda_b200.inference import fold_batchnorm, quantize_linear
    torch.manual_seed(11)
    net = resnet.resnet20().to(DEV)
    images, new = (torch.randn(4, 3, 32, 32, device=DEV) for _ in range(2))
    with torch.no_grad():
        for m in net.modules():
            if isinstance(m, torch.nn.BatchNorm2d):
                m.momentum = 1.0
        net.train()(images)
        for prepare in (fold_batchnorm, quantize_linear):
            prepare(net)
            traced = torch.jit.trace(net, images, check_trace=False)
            assert torch.equal(traced(new), net(new))
