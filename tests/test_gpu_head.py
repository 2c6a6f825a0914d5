"""The operators around a model's head together, as they are used: norm in 8 bits, product to the vocabulary, a teacher's best classes, a student's
step on them, and the check of a student's drafts against the teacher."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_serving_and_training_around_a_head():
    from addernetcuda_b200.distill import DistillationLoss
    from addernetcuda_b200.drafts import verify_drafts
    from addernetcuda_b200.linear8 import linear_8bit, quantize_weight
    from addernetcuda_b200.logprobs import token_log_probs
    from addernetcuda_b200.optim import AdamW
    from addernetcuda_b200.rmsnorm import FusedRMSNorm, rms_norm_8bit
    torch.manual_seed(0)
    d, vocabulary, b, k = 512, 2000, 6, 4
    norm = FusedRMSNorm(d).to(DEV).bfloat16()
    head = torch.randn(vocabulary, d, device=DEV) / d ** 0.5 * 3
    head8 = quantize_weight(head)
    x, stream = (torch.randn(b, k + 1, d, device=DEV).bfloat16() for _ in range(2))
    with torch.no_grad():
        y, h = norm(x, residual=stream, eight=True)
        logits = linear_8bit(y, head8, dtype=torch.float32)
    hd = (x.double() + stream.double()).bfloat16().double()
    exact = hd / (hd.square().mean(-1, keepdim=True) + 2.0 ** -7).sqrt() @ head.double().t()      # an eps of None is bfloat16's
    assert torch.equal(h.double(), hd)
    assert (logits.double() - exact).norm() / exact.norm() < 2 * 2.0 ** -4      # two factors, each within half a step of e4m3

    # a student learns the teacher's best classes at these positions
    best = token_log_probs(logits, top_k=8)
    labels = best.top_indices[..., 0].clone()
    labels[0, 0] = -100
    student_norm = FusedRMSNorm(d).to(DEV)
    student = (0.02 * torch.randn(vocabulary, d, device=DEV)).requires_grad_()
    opt = AdamW([student, *student_norm.parameters()], lr=1e-2)
    loss_of = DistillationLoss(2.0, 0.8)
    inputs = h.float()
    for _ in range(3):
        opt.zero_grad()
        out = student_norm(inputs) @ student.t()
        loss = loss_of(out, labels, best.top_log_probs, best.top_indices)
        loss.backward()
        grads = [p.grad.clone() for p in (student, student_norm.weight)]
        before = [p.detach().clone() for p in (student, student_norm.weight)]
        opt.step()
    ps, pw = (t.double().requires_grad_() for t in before)
    hn = inputs.double()
    out = hn / (hn.square().mean(-1, keepdim=True) + torch.finfo(torch.float32).eps).sqrt() * pw @ ps.t()
    log_t = torch.log_softmax(best.top_log_probs.double() / 2, -1)
    kl = (log_t.exp() * (log_t - torch.log_softmax(out / 2, -1).gather(-1, best.top_indices))).sum(-1)
    nll = -torch.log_softmax(out, -1).gather(-1, labels.clamp(min=0)[..., None])[..., 0]
    counts = labels != -100
    ref = ((0.8 * 4 * kl + 0.2 * nll) * counts).sum() / counts.sum()
    assert abs(loss.double() - ref) <= 1e-4 * abs(ref)
    for got, want in zip(grads, torch.autograd.grad(ref, (ps, pw))):
        assert (got.double() - want).norm() <= 1e-3 * want.norm()

    # its drafts, checked
    with torch.no_grad():
        q = torch.softmax((student_norm(inputs) @ student.t())[:, :k], -1)
        p = torch.softmax(logits, -1)
        drafts = torch.multinomial(q.view(b * k, -1), 1).view(b, k)
        r = verify_drafts(p, q, drafts, torch.rand(b, k + 1, device=DEV))
    for s in range(b):
        n = int(r.accepted[s])
        assert torch.equal(r.tokens[s, :n], drafts[s, :n]) and 0 <= r.tokens[s, n] < vocabulary and (r.tokens[s, n + 1:] == -1).all()
