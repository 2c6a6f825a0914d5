"""Verification of drafts against the definition in float64 (numpy): whole numbers, equal to the last one."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _inputs(b, k, v, dtype, seed=0, sharp=2.5):
    torch.manual_seed(seed)
    logits = sharp * torch.randn(b, k + 1, v, device=DEV)
    p = torch.softmax(logits, -1).to(dtype)
    q = torch.softmax(logits[:, :k] + torch.randn(b, k, v, device=DEV), -1).to(dtype)
    tokens = torch.multinomial(q.float().view(b * k, v), 1).view(b, k) if k else torch.zeros(b, 0, dtype=torch.int64, device=DEV)
    return p, q, tokens, torch.rand(b, k + 1, device=DEV)


def _definition(p, q, tokens, u, lengths=None):
    p, u, tokens = p.double().cpu().numpy(), u.double().cpu().numpy(), tokens.cpu().numpy()
    q = None if q is None else q.double().cpu().numpy()
    b, places, v = p.shape
    out, accepted = np.full((b, places), -1), np.zeros(b, int)
    with np.errstate(invalid="ignore"):
        for s in range(b):
            length = places - 1 if lengths is None else int(np.clip(lengths[s].item(), 0, places - 1))
            n = 0
            while n < length:
                t = tokens[s, n]
                if not (0 <= t < v and u[s, n] * (1.0 if q is None else q[s, n, t]) < p[s, n, t]):
                    break
                out[s, n] = t
                n += 1
            accepted[s] = n
            w = p[s, n].copy()
            if n < length:
                if q is not None:
                    w = w - q[s, n]
                elif 0 <= tokens[s, n] < v:
                    w[tokens[s, n]] = 0
            w = np.where(w > 0, w, 0)
            if not w.sum() > 0:
                w = np.where(p[s, n] > 0, p[s, n], 0)
            total = w.sum()
            if not total > 0 or not np.isfinite(total):
                continue
            reached = np.cumsum(w)
            hits = np.nonzero((reached > u[s, -1] * reached[-1]) & (w > 0))[0]
            out[s, n] = hits[0] if len(hits) else np.nonzero(w > 0)[0][-1]
    return out, accepted


def _check(p, q, tokens, u, lengths=None):
    from addernetcuda_b200.drafts import verify_drafts
    r = verify_drafts(p, q, tokens, u, lengths)
    out, accepted = _definition(p, q, tokens, u, lengths)
    assert np.array_equal(r.accepted.cpu().numpy(), accepted)
    assert np.array_equal(r.tokens.cpu().numpy(), out), (r.tokens.cpu().numpy()[(r.tokens.cpu().numpy() != out).any(1)], out[(r.tokens.cpu().numpy() != out).any(1)])
    return r


@pytest.mark.parametrize("b,k,v", [(1, 1, 1), (1, 4, 32000), (3, 2, 7), (5, 8, 1000), (64, 3, 1001), (2, 40, 500), (7, 5, 50257), (33, 2, 4099), (300, 4, 4096), (16, 3, 20001),
                                   (2, 1, 128000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("certain", [False, True])
def test_by_definition(b, k, v, dtype, certain):
    p, q, tokens, u = _inputs(b, k, v, dtype, seed=b + v)
    if certain:
        tokens = torch.where(torch.rand(b, k, device=DEV) < 0.7, p[:, :k].float().argmax(-1), tokens)
    lengths = torch.randint(-1, k + 2, (b,), device=DEV)
    for chosen in (None, lengths, lengths.int()):
        _check(p, None if certain else q, tokens, u, chosen)


def test_no_drafts():
    p, q, tokens, u = _inputs(9, 0, 5000, torch.float32)
    _check(p, q, tokens, u)
    _check(p, None, tokens, u)


def test_borders():
    """Numbers at the borders: u of 0 and just below 1, weights of 0 before and behind, one class alone, equal probabilities."""
    v = 3000
    p = torch.zeros(6, 2, v, device=DEV)
    q = torch.zeros(6, 1, v, device=DEV)
    p[0, :, 700] = 1.0
    p[1, :, 5] = 0.5
    p[1, :, 2900] = 0.5
    p[2] = 1.0 / v
    p[3, 0, 10] = 0.25
    q[3, 0, 10] = 0.25                 # nothing of the difference is left where it is refused: p itself
    p[4, :, 100] = 0.5
    p[4, :, 200] = 0.5
    q[:, 0, 0] = 1.0
    q[3, 0, 0] = 0.0
    for first in (0.0, 0.999999, 1.0):
        for last in (0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24, 1.0, 1.5, float("nan")):
            u = torch.tensor([first, last], device=DEV).expand(6, 2)
            tokens = torch.tensor([[700], [5], [2999], [10], [200], [3]], device=DEV)
            r = _check(p, q, tokens, u)
            assert r.tokens[5, int(r.accepted[5])] == -1      # no class has a weight
            _check(p, None, tokens, u)


def test_special_values():
    p, q, tokens, u = _inputs(8, 2, 4100, torch.float32, seed=2)
    tokens[0, 0] = -1
    tokens[1, 0] = 4100
    tokens[2, 1] = 2 ** 40
    p[3, :, 7] = float("nan")
    q[4, :, ::2] = float("nan")
    p[5] = 0
    p[6, :, 9] = float("inf")
    q[7] = 2 * p[7, :2]                 # above p everywhere
    u[6] = 0.5
    r = _check(p, q, tokens, u)
    assert r.accepted[0] == 0 and r.accepted[1] == 0 and r.tokens[5, 0] == -1
    _check(p, None, tokens, u)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scale", [1e-3, 3.0, 200.0])
def test_weights_that_are_no_probabilities(dtype, scale):
    """Sums far below and above 1, and single weights of several."""
    for v in (37, 5000, 40001):
        torch.manual_seed(v)
        p = (scale * torch.rand(12, 3, v, device=DEV)).to(dtype)
        q = (scale * torch.rand(12, 2, v, device=DEV)).to(dtype)
        tokens = torch.randint(0, v, (12, 2), device=DEV)
        _check(p, q, tokens, torch.rand(12, 3, device=DEV))
        _check(p, None, tokens, torch.rand(12, 3, device=DEV))


def test_views_and_places_behind_the_length():
    from addernetcuda_b200.drafts import verify_drafts
    p, q, tokens, u = _inputs(6, 3, 1024, torch.bfloat16, seed=3)
    want = _check(p, q, tokens, u)
    wide_p = torch.full((6, 5, 1100), float("nan"), device=DEV, dtype=torch.bfloat16)
    wide_q = torch.full((3, 6, 1030), float("nan"), device=DEV, dtype=torch.bfloat16)
    wide_p[:, :4, 3:1027] = p
    wide_q[..., 1:1025] = q.transpose(0, 1)
    flip = torch.empty(4, 6, device=DEV).t()
    flip.copy_(u)
    got = verify_drafts(wide_p[:, :4, 3:1027], wide_q.transpose(0, 1)[..., 1:1025], tokens.t().contiguous().t(), flip)
    assert torch.equal(got.tokens, want.tokens) and torch.equal(got.accepted, want.accepted)
    got = verify_drafts(p.transpose(1, 2).contiguous().transpose(1, 2), q, tokens.int(), u)
    assert torch.equal(got.tokens, want.tokens)
    lengths = torch.tensor([0, 1, 2, 3, 1, 0], device=DEV)
    want = _check(p, q, tokens, u, lengths)
    p2, q2, t2, u2 = p.clone(), q.clone(), tokens.clone(), u.clone()
    for s, n in enumerate(lengths.tolist()):
        p2[s, n + 1:] = float("nan")
        q2[s, n:] = float("nan")
        t2[s, n:] = 10 ** 9
        u2[s, n:3] = float("nan")
    got = verify_drafts(p2, q2, t2, u2, lengths)
    assert torch.equal(got.tokens, want.tokens) and torch.equal(got.accepted, want.accepted)


def test_tokens_are_distributed_as_the_target():
    """The first token of many sequences: chi-square of 20 classes below its value for one chance in a million."""
    b, v = 200000, 20
    torch.manual_seed(4)
    p = torch.softmax(torch.randn(2, v, device=DEV), -1)
    q = torch.softmax(torch.randn(1, v, device=DEV), -1)
    tokens = torch.multinomial(q[0], b, replacement=True).view(b, 1)
    from addernetcuda_b200.drafts import verify_drafts
    r = verify_drafts(p.expand(b, 2, v), q.expand(b, 1, v), tokens, torch.rand(b, 2, device=DEV))
    seen = torch.bincount(r.tokens[:, 0], minlength=v).double()
    expected = p[0].double() * b
    assert ((seen - expected) ** 2 / expected).sum() < 66.7
    share = torch.minimum(p[0], q[0]).sum().item()
    assert abs(r.accepted.double().mean().item() - share) < 5 * (0.25 / b) ** 0.5


def test_captured_on_another_stream_and_two_at_once():
    from addernetcuda_b200.drafts import verify_drafts
    cases = [_inputs(b, k, v, torch.bfloat16, seed=v) for b, k, v in ((2, 3, 40000), (64, 4, 5000))]
    want = [verify_drafts(*c) for c in cases]
    graphs = []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = verify_drafts(*c)
        graphs.append((g, r))
    streams = [torch.cuda.Stream() for _ in cases]
    for (g, r), s in zip(graphs, streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(3):
                g.replay()
    torch.cuda.synchronize()
    for (g, r), w in zip(graphs, want):
        assert torch.equal(r.tokens, w.tokens) and torch.equal(r.accepted, w.accepted)


def test_offsets_beyond_32_bits():
    b, k, v = 2, 16, 70_000_000
    p = torch.zeros(b, k + 1, v, dtype=torch.bfloat16, device=DEV)
    p[:, :, -1] = 0.5
    p[:, :, -70_000] = 0.5
    q = torch.zeros(1, 1, v, dtype=torch.bfloat16, device=DEV)
    q[..., -1] = 1.0
    tokens = torch.full((b, k), v - 1, device=DEV)
    u = torch.full((b, k + 1), 0.25, device=DEV)
    u[1, k - 1] = 0.75
    from addernetcuda_b200.drafts import verify_drafts
    r = verify_drafts(p, q.expand(b, k, v), tokens, u)
    assert r.accepted.tolist() == [k, k - 1] and r.tokens[0, k] == v - 70_000 and r.tokens[1, k - 1] == v - 70_000 and r.tokens[1, k] == -1


def test_refusals():
    from addernetcuda_b200.drafts import verify_drafts
    p, q, tokens, u = _inputs(3, 2, 50, torch.float32)
    lengths = torch.ones(3, dtype=torch.int64, device=DEV)
    for bad, kind in ((lambda: verify_drafts(p[0], q, tokens, u), ValueError), (lambda: verify_drafts(p, q[:, :1], tokens, u), ValueError),
                      (lambda: verify_drafts(p, q.half(), tokens, u), ValueError), (lambda: verify_drafts(p, q, tokens[:, :1], u), ValueError),
                      (lambda: verify_drafts(p, q, tokens.float(), u), TypeError), (lambda: verify_drafts(p, q, tokens, u[:, :2]), ValueError),
                      (lambda: verify_drafts(p, q, tokens, u.double()), TypeError), (lambda: verify_drafts(p, q, tokens, u, lengths[:2]), ValueError),
                      (lambda: verify_drafts(p, q, tokens.cpu(), u), RuntimeError), (lambda: verify_drafts(p.cpu(), q, tokens, u), RuntimeError),
                      (lambda: verify_drafts(p[:, :0], q, tokens, u), ValueError), (lambda: verify_drafts(p.double(), q, tokens, u), TypeError)):
        with pytest.raises(kind):
            bad()
    assert verify_drafts(p[:0], q[:0], tokens[:0], u[:0]).tokens.shape == (0, 3)
