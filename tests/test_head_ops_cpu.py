"""RMS norm, the product in 8 bits, distillation and the verification of drafts without a GPU: what the C interface and the Python
layer refuse."""
import pytest
import torch

P = 4096      # stands for a pointer that no refused call follows
NULL, SHAPE, UNSUPPORTED, ALIGNMENT, WORKSPACE = 1, 2, 3, 4, 5


def _lib():
    from addernetcuda_b200 import _lib
    return _lib.load()


def _caller(name, **defaults):
    entry = getattr(_lib(), name)
    return lambda **k: entry(*{**defaults, **k}.values())


def test_rms_norm():
    call = _caller("adder_b200_rmsnorm_forward", x=P, r=None, w=P, y=P, h=None, rstd=None, rows=2, d=8, xs=8, rs=0, t=0, wt=0, eps=1e-6, s=None)
    assert call(rows=0) == 0
    for k in (dict(rows=-1), dict(d=0), dict(eps=-1.0), dict(eps=float("nan")), dict(xs=-8), dict(rs=-1)):
        assert call(**k) == SHAPE
    for k in (dict(t=3), dict(t=1, wt=2), dict(wt=1), dict(d=1 << 40), dict(rows=1 << 31)):
        assert call(**k) == UNSUPPORTED
    assert call(x=None) == call(y=None) == call(r=P) == NULL
    assert call(x=P + 2) == call(t=1, w=P + 2) == call(rstd=P + 2) == ALIGNMENT
    eight = _caller("adder_b200_rmsnorm_forward_8bit", x=P, r=None, w=P, v=P, sc=P, h=None, rows=2, d=8, xs=8, rs=0, vs=16, t=0, wt=0, eps=1e-6, s=None)
    assert eight(rows=0) == 0 and eight(vs=7) == eight(d=0) == eight(eps=-1.0) == SHAPE
    assert eight(v=None) == eight(sc=None) == eight(x=None) == eight(r=P) == NULL and eight(sc=P + 1) == eight(h=P + 1) == ALIGNMENT and eight(t=9) == UNSUPPORTED
    back = _caller("adder_b200_rmsnorm_backward", dy=P, dh=None, h=P, w=P, rstd=P, dx=P, dw=P, ws=P, bytes=1 << 20, rows=2, d=8, hs=8, t=0, wt=0, s=None)
    assert back(d=0) == back(hs=-1) == SHAPE and back(t=9) == UNSUPPORTED and back(dy=None) == back(h=None) == back(rstd=None) == NULL
    assert back(dx=P + 1) == back(ws=P + 4) == ALIGNMENT and back(ws=None) == back(bytes=8) == WORKSPACE and back(dx=None, dw=None) == 0
    size = _lib().adder_b200_rmsnorm_backward_workspace_bytes
    assert size(0, 8) == size(2, 0) == 0 and size(4, 8) >= 8 * 4


def test_products_in_8_bits():
    for name in ("rows", "weight"):
        quant = _caller(f"adder_b200_quantize_{name}", x=P, v=P, sc=P, rows=2, d=8, xs=8, vs=16, t=0, s=None)
        assert quant(rows=0) == 0 and quant(rows=-1) == quant(d=0) == quant(vs=7) == quant(xs=-1) == SHAPE and quant(t=3) == quant(d=1 << 33, vs=1 << 33) == UNSUPPORTED
        assert quant(x=None) == quant(v=None) == quant(sc=None) == NULL and quant(x=P + 2) == quant(t=1, x=P + 1) == quant(sc=P + 2) == ALIGNMENT
    call = _caller("adder_b200_linear_8bit", x=P, xs=P, w=P, ws=P, b=None, y=P, m=4, k=100, n=8, xst=112, wst=112, t=1, s=None)
    assert call(m=0) == call(n=0) == 0
    assert call(m=-1) == call(k=0) == call(n=-1) == call(xst=99) == call(wst=96) == SHAPE
    assert call(t=4) == call(m=1 << 32) == call(n=1 << 32) == call(k=1 << 32, xst=1 << 32, wst=1 << 32) == UNSUPPORTED
    for name in ("x", "xs", "w", "ws", "y"):
        assert call(**{name: None}) == NULL
    assert call(x=P + 8) == call(w=P + 1) == call(xst=104) == call(wst=120) == call(y=P + 1) == call(b=P + 1) == call(xs=P + 2) == ALIGNMENT


def test_distillation():
    fwd = _caller("adder_b200_distillation_forward", x=P, t=0, rows=2, v=10, xs=10, z=P, zt=0, at=P, k=3, tau=1.0, tg=None, ig=-100, d=P, lp=None, st=None, ma=None, s=None)
    assert fwd(rows=0) == 0
    assert fwd(rows=-1) == fwd(v=0) == fwd(k=0) == fwd(tau=0.0) == fwd(tau=-1.0) == fwd(tau=float("inf")) == fwd(tau=float("nan")) == fwd(xs=-1) == SHAPE
    assert fwd(k=257) == fwd(t=3) == fwd(zt=-1) == fwd(v=1 << 31) == fwd(rows=1 << 30) == UNSUPPORTED
    assert fwd(x=None) == fwd(z=None) == fwd(at=None) == fwd(d=None) == fwd(tg=P) == fwd(lp=P) == fwd(st=P) == fwd(ma=P) == NULL
    assert fwd(x=P + 2) == fwd(t=1, x=P + 1) == fwd(z=P + 2) == fwd(at=P + 4) == fwd(d=P + 2) == fwd(tg=P + 4, lp=P) == ALIGNMENT
    bwd = _caller("adder_b200_distillation_backward", x=P, t=0, rows=2, v=10, xs=10, at=P, k=3, tau=1.0, tg=None, ig=-100, st=P, ma=P, gd=P, gl=None, dx=P, s=None)
    assert bwd(rows=0) == 0 and bwd(k=0) == bwd(tau=0.0) == SHAPE and bwd(k=300) == bwd(t=7) == UNSUPPORTED
    assert bwd(st=None) == bwd(ma=None) == bwd(dx=None) == bwd(at=None) == bwd(gl=P) == NULL
    assert bwd(dx=P + 2) == bwd(gd=P + 1) == bwd(st=P + 2) == ALIGNMENT


def test_verification_of_drafts():
    call = _caller("adder_b200_verify_drafts", p=P, q=P, t=0, tk=P, u=P, ln=None, out=P, acc=P, b=2, k=3, v=10, ps=40, pp=10, qs=30, qp=10, s=None)
    assert call(b=0) == 0
    assert call(b=-1) == call(k=-1) == call(v=0) == call(ps=-1) == call(pp=-1) == call(qs=-1) == call(qp=-1) == SHAPE
    assert call(t=3) == call(v=1 << 31) == call(k=65536) == call(b=1 << 30) == UNSUPPORTED
    assert call(p=None) == call(tk=None) == call(u=None) == call(out=None) == call(acc=None) == NULL
    assert call(p=P + 2) == call(q=P + 2) == call(tk=P + 4) == call(u=P + 2) == call(ln=P + 4) == call(out=P + 4) == call(acc=P + 4) == ALIGNMENT


def test_python_layer_refuses_what_is_not_on_a_gpu():
    from addernetcuda_b200.distill import DistillationLoss, distillation
    from addernetcuda_b200.drafts import verify_drafts
    from addernetcuda_b200.linear8 import Rows8, Weight8, linear_8bit, quantize_rows, quantize_weight
    from addernetcuda_b200.rmsnorm import FusedRMSNorm, rms_norm, rms_norm_8bit
    x = torch.randn(4, 8)
    at = torch.zeros(4, 2, dtype=torch.int64)
    codes = Rows8(x.to(torch.float8_e4m3fn), torch.ones(4, 1)), Weight8(x.to(torch.float8_e4m3fn), torch.ones(1, 1))
    for call in (lambda: rms_norm(x, 8), lambda: rms_norm_8bit(x), lambda: quantize_rows(x), lambda: quantize_weight(x), lambda: linear_8bit(*codes),
                 lambda: linear_8bit(x, codes[1]), lambda: distillation(x, x[:, :2], at), lambda: verify_drafts(x.view(2, 2, 8), None, at[:2, :1], torch.rand(2, 2)),
                 lambda: FusedRMSNorm(8)(x, eight=True)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    for call in (lambda: rms_norm([1.0], 1), lambda: rms_norm_8bit(3), lambda: linear_8bit(x, x), lambda: distillation(None, x, at), lambda: verify_drafts(1, 2, 3, 4)):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(ValueError):
        DistillationLoss(alpha=-0.1)


def test_norm_on_the_cpu_goes_through_torch():
    from addernetcuda_b200.rmsnorm import FusedRMSNorm
    x, r = torch.randn(4, 8), torch.randn(4, 8)
    m = FusedRMSNorm(8)
    assert torch.equal(m(x), torch.nn.functional.rms_norm(x, (8,), m.weight))
    y, h = m(x, residual=r)
    assert torch.equal(h, x + r) and torch.equal(y, torch.nn.functional.rms_norm(h, (8,), m.weight))


def test_values_of_codes():
    from addernetcuda_b200.linear8 import Rows8, Weight8
    torch.manual_seed(0)
    codes, xs, ws = torch.randn(130, 200).to(torch.float8_e4m3fn), torch.rand(130, 2), torch.rand(2, 2)
    x, w = Rows8(codes, xs).dequantize(), Weight8(codes, ws).dequantize(torch.float64)
    for i, j in ((0, 0), (127, 127), (128, 128), (129, 199), (3, 130)):
        assert x[i, j] == codes[i, j].float() * xs[i, j // 128] and w[i, j] == (codes[i, j].float() * ws[i // 128, j // 128]).double()
