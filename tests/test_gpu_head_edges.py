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
