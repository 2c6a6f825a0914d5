"""The operators together, as they are used: a step of a small token network of adder columns - norms with a residual stream, logits,
loss, backward, AdamW - against the same network in float64, captured as a graph, and inside the training step of this package."""
import pytest
import torch
import torch.nn as nn

from addernetcuda_b200 import adder as A
from addernetcuda_b200.layernorm import FusedLayerNorm
from addernetcuda_b200.logprobs import TokenCrossEntropy, token_log_probs
from addernetcuda_b200.optim import AdamW
from addernetcuda_b200.train import TrainStep

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class Tokens(nn.Module):
    """h = embedding; h += mix(norm(h)) twice; logits of norm(h)."""

    def __init__(self, vocabulary=97, width=48, adders=True):
        super().__init__()
        self.embed = nn.Embedding(vocabulary, width)
        make = (lambda: A.adder2d(width, width, 1)) if adders else (lambda: nn.Conv2d(width, width, 1, bias=False))
        self.mix = nn.ModuleList([make() for _ in range(2)])
        self.norms = nn.ModuleList([FusedLayerNorm(width) for _ in range(3)])
        self.head = nn.Linear(width, vocabulary, bias=False)

    def forward(self, tokens):
        h = self.embed(tokens)
        y = self.norms[0](h)
        for mix, norm in zip(self.mix, self.norms[1:]):
            d = mix(y.transpose(1, 2).unsqueeze(2)).squeeze(2).transpose(1, 2) * 0.05
            y, h = norm(d, residual=h)
        return self.head(y)


def _batch(seed, n=4, length=13, vocabulary=97):
    torch.manual_seed(seed)
    t = torch.randint(0, vocabulary, (n, length + 1), device=DEV)
    inputs, targets = t[:, :-1].contiguous(), t[:, 1:].clone()
    targets[0, length // 2:] = -100      # a padded sequence
    return inputs, targets


def _reference(model, tokens, targets):
    """The same formulas in float64 with plain operations (multiply-based mixing)."""
    p = {k: v.detach().double().requires_grad_() for k, v in model.named_parameters()}

    def norm(h, i):
        c = h - h.mean(-1, keepdim=True)
        return c / (c.square().mean(-1, keepdim=True) + 1e-5).sqrt() * p[f"norms.{i}.weight"] + p[f"norms.{i}.bias"]

    h = p["embed.weight"][tokens]
    y = norm(h, 0)
    for i in range(2):
        h = h + y @ p[f"mix.{i}.weight"][:, :, 0, 0].t() * 0.05
        y = norm(h, i + 1)
    logp = torch.log_softmax(y @ p["head.weight"].t(), -1)
    given = targets != -100
    loss = -logp.gather(-1, torch.where(given, targets, 0)[..., None])[..., 0][given].mean()
    loss.backward()
    return loss.detach(), {k: v.grad for k, v in p.items()}


def test_a_step_against_float64():
    torch.backends.cuda.matmul.allow_tf32 = torch.backends.cudnn.allow_tf32 = False
    torch.manual_seed(0)
    model = Tokens(adders=False).to(DEV)
    opt = AdamW(model.parameters(), lr=1e-2)
    loss_of = TokenCrossEntropy()
    for step in range(3):
        tokens, targets = _batch(step)
        want_loss, want = _reference(model, tokens, targets)
        opt.zero_grad()
        loss = loss_of(model(tokens), targets)
        loss.backward()
        # fp32 products and sums of 48 to 97 terms through three layers: some 500 roundings of 2^-24 relative to the largest gradient
        assert abs(float(loss) - float(want_loss)) <= 500 * 2.0 ** -24 * (1 + float(want_loss))
        for k, q in model.named_parameters():
            scale = max(float(want[k].abs().max()), 1e-3)
            assert float((q.grad.double() - want[k]).abs().max()) <= 2000 * 2.0 ** -24 * scale, k
        opt.step()


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_training_of_an_adder_network_equals_the_eager_one(bits):
    def build():
        torch.manual_seed(1)
        model = Tokens().to(DEV)
        return model, AdamW(model.parameters(), lr=1e-2, state_bits=bits, min_8bit_size=1024), TokenCrossEntropy()

    def step(model, opt, loss_of, tokens, targets):
        opt.zero_grad(set_to_none=True)
        loss = loss_of(model(tokens), targets)
        loss.backward()
        opt.step()
        return loss.detach()

    eager, captured = build(), build()
    tokens, targets = _batch(0)
    ts, gs = tokens.clone(), targets.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*captured, ts, gs)
    torch.cuda.current_stream().wait_stream(side)
    step(*eager, tokens, targets)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = step(*captured, ts, gs)
    for i in range(1, 4):
        tokens, targets = _batch(i)
        ts.copy_(tokens); gs.copy_(targets)
        graph.replay()
        want = step(*eager, tokens, targets)
        # torch's own products and scatters may add up in another order under capture: 1e-6, which a step of AdamW can turn into a
        # learning rate (1e-2) where a gradient is rounding noise; such weights move the loss of 100 tokens by far less
        assert abs(float(loss) - float(want)) <= 1e-2 * float(want)
    for p in captured[0].parameters():
        assert bool(p.isfinite().all())
    for opt in (captured[1], eager[1]):
        assert all(int(s["step"][0]) == 4 and int(s["step"][1]) == 0 for s in opt.state.values())


def test_sampling_from_the_network():
    torch.manual_seed(2)
    model = Tokens().to(DEV).eval()
    with torch.no_grad():
        tokens, _ = _batch(0)
        for _ in range(3):
            logits = model(tokens)[:, -1]               # rows of a larger buffer
            r = token_log_probs(logits, top_k=5, entropy=True)
            assert torch.equal(r.top_indices[:, 0], logits.argmax(-1))
            p = torch.log_softmax(logits.double(), -1)
            assert float((r.top_log_probs.double() - p.gather(1, r.top_indices)).abs().max()) < 1e-5
            tokens = torch.cat([tokens, r.top_indices[:, :1]], 1)


@pytest.mark.parametrize("optimizer", ["adamw", "adamw8"])
def test_training_step_with_own_loss_and_optimizer(optimizer):
    from addernetcuda_b200 import resnet as R
    rows = {}
    for use_graph in (False, True):
        torch.manual_seed(0)
        net = R.resnet20().to(DEV)
        R.init_seeded(net, 0)
        ts = TrainStep(net, (16, 3, 32, 32), 10, lr=1e-3, use_graph=use_graph, device=DEV, optimizer=optimizer, criterion=TokenCrossEntropy())
        losses = []
        for i in range(3):
            torch.manual_seed(i)
            loss = ts.step(torch.randn(16, 3, 32, 32, device=DEV), torch.randint(0, 10, (16,), device=DEV))
            losses.append(loss.item())
        assert all(l == l and l < 20 for l in losses)
        rows[use_graph] = ts
    eager, graph = rows[False], rows[True]
    n = lambda ts: int(next(iter(ts.opt.state.values()))["step"][0])      # noqa: E731
    assert n(eager) == 3 and n(graph) == 3 + 3      # three warm-up steps before the capture
    with pytest.raises(ValueError, match="optimizer"):
        TrainStep(R.resnet20().to(DEV), (2, 3, 32, 32), 10, device=DEV, optimizer="lion")


def test_loss_and_accuracy_of_an_evaluation():
    from addernetcuda_b200 import resnet as R
    from addernetcuda_b200.inference import evaluate, fold_batchnorm, validate
    net = R.resnet20().to(DEV)
    R.init_seeded(net, 0)
    net = fold_batchnorm(net)
    torch.manual_seed(0)
    batches = [(torch.randn(n, 3, 32, 32), torch.randint(0, 10, (n,))) for n in (8, 5)]
    got = evaluate(batches, net, DEV, topk=(1, 5))
    assert got["topk"] == pytest.approx(validate(batches, net, DEV, topk=(1, 5)))
    with torch.no_grad():
        logp = torch.cat([torch.log_softmax(net(x.to(DEV)).double(), 1) for x, _ in batches])
    labels = torch.cat([y for _, y in batches]).to(DEV)
    assert got["loss"] == pytest.approx(float(-logp.gather(1, labels[:, None]).mean()), rel=1e-5)
    assert got["entropy"] == pytest.approx(float(-(logp.exp() * logp).sum(1).mean()), rel=1e-5, abs=1e-6)


class Classifier(torch.nn.Module):
    """A norm and a product of this library's and elementwise operations, whose sums have one order: the same bits in every run.  63 columns, so
    that gradients one behind another in a bucket do not begin at 16 bytes."""

    def __init__(self):
        super().__init__()
        gen = torch.Generator()
        gen.manual_seed(5)
        self.norm = FusedLayerNorm(63)
        self.scale = torch.nn.Parameter(0.3 * torch.randn(67, 63, generator=gen))
        self.shift = torch.nn.Parameter(torch.zeros(67))

    def forward(self, x):
        return (self.norm(x)[:, None] * self.scale).sum(-1) + self.shift


@pytest.mark.parametrize("optimizer", ["adamw", "adamw8"])
def test_training_steps_captured_or_not_and_with_gradients_in_buckets_give_the_same_bits(optimizer, tmp_path):
    import torch.distributed as dist
    from addernetcuda_b200.ddp import BucketedDDP

    def train(use_graph, with_ddp):
        net = Classifier().to(DEV)
        ddp = BucketedDDP(net) if with_ddp else None
        ts = TrainStep(net, (24, 63), 67, lr=3e-3, weight_decay=0.01, ddp=ddp, use_graph=use_graph, device=DEV, optimizer=optimizer, criterion=TokenCrossEntropy())
        gen = torch.Generator(device=DEV)
        gen.manual_seed(6)
        losses = []
        for i in range(4):
            x, y = torch.randn(24, 63, device=DEV, generator=gen), torch.randint(0, 67, (24,), device=DEV, generator=gen)
            for _ in range(1 if use_graph or i else 4):      # a captured step is preceded by three eager ones on the first batch
                losses.append(ts.step(x, y).clone())
        if with_ddp:
            assert any(p.grad.data_ptr() % 16 for p in net.parameters())
        assert all(s["step"].tolist() == [7, 0] for s in ts.opt.state.values())
        states = [s[k] for s in ts.opt.state.values() for k in ("exp_avg", "exp_avg_sq")]
        assert optimizer == "adamw" or any(t.dtype == torch.uint8 for t in states)
        return losses[-4:], [p.detach() for p in net.parameters()] + states

    dist.init_process_group("gloo", init_method=f"file://{tmp_path}/store", rank=0, world_size=1)
    try:
        runs = [train(use_graph, with_ddp) for with_ddp in (False, True) for use_graph in (False, True)]
    finally:
        dist.destroy_process_group()
    assert float(runs[0][0][-1]) != float(runs[0][0][-2])
    for losses, tensors in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(losses, runs[0][0]))
        assert all(torch.equal(a, b) for a, b in zip(tensors, runs[0][1]))


def test_a_label_that_is_no_class_is_no_hit_on_a_row_without_classes():
    from addernetcuda_b200.inference import evaluate
    logits = torch.tensor([[1.0, 2.0, 3.0], [float("nan"), 0.0, 0.0], [5.0, 1.0, 0.0], [0.0, 9.0, 1.0]])
    got = evaluate([(logits, torch.tensor([2, -1, 0, -100]))], torch.nn.Identity(), DEV, topk=(1, 2))
    assert got["topk"] == pytest.approx((200 / 3, 200 / 3)) and got["loss"] != got["loss"]
