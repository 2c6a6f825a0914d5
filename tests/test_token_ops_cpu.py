"""Layer norm, log probabilities and AdamW without a GPU: what the C interface and the Python layer refuse, and the
8-bit format's arithmetic against its definition."""
import ctypes

import numpy as np
import pytest
import torch


def _lib():
    from addernetcuda_b200 import _lib
    return _lib.load()


P = 4096      # stands for a pointer that no refused call follows


def test_layer_norm_entry_points_check_their_arguments():
    lib = _lib()
    call = lambda **k: lib.adder_b200_layernorm_forward(*({**dict(x=P, r=None, w=P, b=P, y=P, h=None, mean=None, rstd=None, rows=2, d=8,
                                                                  xs=8, rs=0, t=0, wt=0, eps=1e-5, s=None), **k}).values())
    assert call(rows=-1) == 2 and call(d=0) == 2 and call(eps=-1.0) == 2 and call(xs=-8) == 2 and call(eps=float("nan")) == 2
    assert call(rows=0) == 0
    assert call(t=3) == 3 and call(t=1, wt=2) == 3 and call(t=0, wt=1) == 3 and call(d=1 << 40) == 3 and call(rows=1 << 31) == 3
    assert call(x=None) == 1 and call(y=None) == 1 and call(r=P) == 1 and call(mean=P) == 1      # residual without h, mean without rstd
    assert call(x=P + 2) == 4 and call(t=1, wt=0, w=P + 2) == 4
    back = lambda **k: lib.adder_b200_layernorm_backward(*({**dict(dy=P, dh=None, h=P, w=P, mean=P, rstd=P, dx=P, dw=P, db=P, ws=P,
                                                                   bytes=1 << 20, rows=2, d=8, hs=8, t=0, wt=0, s=None), **k}).values())
    assert back(d=0) == 2 and back(hs=-1) == 2 and back(t=9) == 3
    assert back(dy=None) == 1 and back(h=None) == 1 and back(mean=None) == 1
    assert back(dx=P + 1) == 4
    assert back(ws=None) == 5 and back(bytes=8) == 5
    assert lib.adder_b200_layernorm_backward_workspace_bytes(0, 8) == 0 and lib.adder_b200_layernorm_backward_workspace_bytes(2, 0) == 0
    assert lib.adder_b200_layernorm_backward_workspace_bytes(4, 8) >= 2 * 8 * 4
    most = 2 ** 30 - 2 ** 16
    assert call(d=most + 1) == back(d=most + 1) == back(d=2 ** 31) == call(d=2 ** 30)
    assert call(d=most + 1) not in (0, call(d=0)) and back(d=most + 1) not in (0, back(d=0))
    assert lib.adder_b200_layernorm_backward_workspace_bytes(1, most + 1) == 0 < lib.adder_b200_layernorm_backward_workspace_bytes(1, most)


def test_log_probs_entry_points_check_their_arguments():
    lib = _lib()
    call = lambda **k: lib.adder_b200_log_probs_forward(*({**dict(x=P, t=0, rows=2, classes=8, stride=8, targets=P, ignore=-100, k=0, lp=P,
                                                                  ent=None, stats=None, top=None, idx=None, s=None), **k}).values())
    assert call(rows=-1) == 2 and call(classes=0) == 2 and call(k=-1) == 2 and call(k=9) == 2 and call(stride=-8) == 2
    assert call(rows=0) == 0
    assert call(t=3) == 3 and call(classes=1 << 40) == 3 and call(k=33, classes=64) == 3
    assert call(x=None) == 1 and call(targets=None) == 1 and call(k=2) == 1
    assert call(x=P + 2) == 4
    back = lambda **k: lib.adder_b200_log_probs_backward(*({**dict(x=P, t=0, rows=2, classes=8, stride=8, targets=P, ignore=-100, k=0,
                                                                   idx=None, stats=P, ent=None, g=P, ge=None, gt=None, dx=P, s=None), **k}).values())
    assert back(classes=0) == 2 and back(k=9) == 2 and back(t=-1) == 3 and back(rows=0) == 0
    assert back(stats=None) == 1 and back(dx=None) == 1 and back(ge=P) == 1 and back(gt=P) == 1 and back(targets=None) == 1
    assert back(dx=P + 1) == 4


def test_adamw_entry_points_check_their_arguments():
    from addernetcuda_b200.optim import _Tensor
    lib = _lib()

    def call(count=1, t=0, bits=32, lr=1e-3, b1=0.9, b2=0.99, eps=1e-8, wd=0.0, null=False, **k):
        f = dict(param=P, grad=P, exp_avg=P, exp_avg_sq=P, exp_avg_scale=None, exp_avg_sq_scale=None, step=P, n=8)
        one = (_Tensor * 1)(_Tensor(*{**f, **k}.values()))
        return lib.adder_b200_adamw_step(None if null else one, count, t, bits, lr, None, b1, b2, eps, wd, None, None)

    assert call(count=-1) == 2 and call(b1=1.0) == 2 and call(b2=-0.1) == 2 and call(eps=-1.0) == 2 and call(lr=float("inf")) == 2
    assert call(wd=float("nan")) == 2 and call(n=-1) == 2 and call(b1=float("nan")) == 2
    assert call(count=0) == 0 and call(n=0) == 0 and call(n=0, param=None) == 0
    assert call(bits=16) == 3 and call(t=7) == 3
    assert call(null=True) == 1 and call(grad=None) == 1 and call(step=None) == 1 and call(bits=8) == 1
    assert call(param=P + 2) == 4 and call(exp_avg=P + 1) == 4 and call(t=1, grad=P + 1) == 4 and call(step=P + 2) == 4
    v = lib.adder_b200_adamw_state_values
    assert v(P, P, 1, P, -1, None) == 2 and v(None, P, 1, P, 8, None) == 1 and v(P, P, 1, P + 2, 8, None) == 4 and v(None, None, 1, None, 0, None) == 0


def test_the_c_struct_is_laid_out_as_the_header_says():
    from addernetcuda_b200.optim import _Tensor
    assert ctypes.sizeof(_Tensor) == 64 and _Tensor.n.offset == 56 and _Tensor.step.offset == 48


def test_cpu_tensors_are_refused():
    from addernetcuda_b200.layernorm import layer_norm
    from addernetcuda_b200.logprobs import TokenCrossEntropy, token_log_probs
    from addernetcuda_b200.optim import AdamW, adamw_state_values, adamw_step
    x = torch.randn(3, 8)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        layer_norm(x, 8)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        token_log_probs(x, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        TokenCrossEntropy()(x, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="must be CUDA tensors"):
        adamw_step([x], [x.clone()], [x.clone()], [x.clone()], torch.zeros(1, 2, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        adamw_state_values(torch.zeros(8, dtype=torch.uint8), torch.zeros(1), True)
    p = torch.nn.Parameter(x)
    p.grad = torch.ones_like(x)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        AdamW([p]).step()


def test_lists_of_different_lengths_and_settings_are_refused():
    from addernetcuda_b200.logprobs import TokenCrossEntropy
    from addernetcuda_b200.optim import AdamW, adamw_step
    x = torch.randn(3)
    with pytest.raises(ValueError, match="grads has 0 tensors, params 1"):
        adamw_step([x], [], [x], [x], [x])
    with pytest.raises(ValueError, match="go together"):
        adamw_step([x], [x], [x], [x], [x], exp_avg_scales=[x])
    adamw_step([], [], [], [], [])      # nothing to do
    p = [torch.nn.Parameter(x)]
    for bad in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1e-8), dict(weight_decay=-0.1), dict(state_bits=16)):
        with pytest.raises(ValueError):
            AdamW(p, **bad)
    with pytest.raises(ValueError):
        TokenCrossEntropy(reduction="median")


def test_layer_norm_module_on_the_cpu_is_torchs():
    from addernetcuda_b200.layernorm import FusedLayerNorm
    m, ref = FusedLayerNorm((4, 3)), torch.nn.LayerNorm((4, 3))
    assert list(m.state_dict()) == list(ref.state_dict())
    x, r = torch.randn(5, 4, 3), torch.randn(5, 4, 3)
    assert torch.equal(m(x), ref(x))
    y, h = m(x, residual=r)
    assert torch.equal(h, x + r) and torch.equal(y, ref(x + r))


@pytest.mark.parametrize("signed,codes", [(True, 128), (False, 256)])
def test_codes_are_the_nearest_of_the_numbers_that_they_stand_for(signed, codes):
    """The rounding of the plain form that the kernels are compared with: magnitudes with 3 (4) exponent and 4 fraction bits, subnormal ones
    at the low end, the code of the nearest magnitude and, half way, the even one."""
    from tests.adamw_plain import decode, encode
    e, f = np.arange(codes) >> 4, np.arange(codes) & 15
    want = np.where(e == 0, f / 16 * 2.0, (1 + f / 16) * 2.0 ** np.maximum(e, 1))
    got = decode(torch.arange(codes, dtype=torch.uint8).repeat(256 // codes), torch.ones(1), signed)[:codes].double().numpy()
    assert np.array_equal(got, want)
    top = 248.0 if signed else 63488.0
    assert want[-1] == top
    rng = np.random.default_rng(3)
    x = np.concatenate([[top], rng.uniform(0, top, 100), 2.0 ** rng.uniform(-5, np.log2(top), 123), (want[1:17] + want[2:18]) / 2, want[:16]])
    x = torch.from_numpy(x[:256].astype(np.float32))
    c, scale = encode(x, signed)
    assert float(scale[0]) == 1.0
    dist = np.abs(x.double().numpy()[:, None] - want[None])
    best = dist.min(1)
    c = c.numpy().astype(int)
    chosen = dist[np.arange(256), c]
    small = (x.numpy() > 0) & (c == 1) if not signed else np.zeros(256, bool)      # never 0 for a second moment that is not
    assert np.array_equal(chosen[~small], best[~small])
    tie = (dist == best[:, None]).sum(1) == 2
    assert tie.sum() >= 10 and np.all(c[tie & ~small] % 2 == 0)


def test_an_eps_below_the_normal_numbers_is_refused():
    """Its reciprocal, where the second moment is 0, is beyond the range."""
    from addernetcuda_b200.optim import AdamW, _Tensor
    lib = _lib()
    call = lambda eps: lib.adder_b200_adamw_step((_Tensor * 1)(_Tensor(P, P, P, P, None, None, P, 0)), 1, 0, 32, 1e-3, None, 0.9, 0.99, eps, 0.0, None, None)      # noqa: E731
    assert call(1e-40) == call(2.0 ** -127) == call(1e-300) == 2 and call(0.0) == call(2.0 ** -126) == 0
    p = [torch.nn.Parameter(torch.zeros(3))]
    with pytest.raises(ValueError, match="eps"):
        AdamW(p, eps=1e-40)
    AdamW(p, eps=0.0), AdamW(p, eps=2.0 ** -126)


def test_the_workspace_of_layer_norm_is_what_its_kernels_write():
    """Rows beyond 8192 elements: sums of the splits of the rows, a small part of the input; shorter ones: sums of every CTA that stays."""
    size = _lib().adder_b200_layernorm_backward_workspace_bytes
    pair = lambda d: 2 * d * 4      # noqa: E731
    assert size(592, 1 << 20) == pair(1 << 20)
    for rows, d in ((64, 50176), (1000, 60000), (600, 1000000), (4096, 8193), (10 ** 6, 16384)):
        assert pair(d) <= size(rows, d) <= max(pair(d), rows * d // 4) and size(rows, d) <= 512 * pair(d)
        assert size(rows, d) % pair(d) == 0 and size(rows, d) // pair(d) <= -(-rows // 32)
    assert size(4, 8192) == 4 * pair(8192) and size(10 ** 6, 8192) >= 128 * pair(8192)


def test_addresses_that_a_type_does_not_allow_are_refused():
    """Targets, outputs, gradients and device scalars: a kernel that follows such an address faults."""
    from addernetcuda_b200.optim import _Tensor
    lib = _lib()
    forward = dict(x=P, t=0, rows=2, classes=8, stride=8, targets=P, ignore=-100, k=2, lp=P, ent=P, stats=P, top=P, idx=P, s=None)
    for name, by in (("targets", 4), ("lp", 2), ("ent", 2), ("stats", 4), ("top", 2), ("idx", 4)):
        assert lib.adder_b200_log_probs_forward(*{**forward, name: P + by}.values()) == 4, name
    backward = dict(x=P, t=0, rows=2, classes=8, stride=8, targets=P, ignore=-100, k=2, idx=P, stats=P, ent=P, g=P, ge=P, gt=P, dx=P, s=None)
    for name, by in (("targets", 4), ("idx", 4), ("stats", 2), ("ent", 2), ("g", 2), ("ge", 2), ("gt", 2)):
        assert lib.adder_b200_log_probs_backward(*{**backward, name: P + by}.values()) == 4, name
    one = (_Tensor * 1)(_Tensor(P, P, P, P, None, None, P, 8))
    for lr, scale in ((P + 2, None), (None, P + 1)):
        assert lib.adder_b200_adamw_step(one, 1, 0, 32, 1e-3, lr, 0.9, 0.99, 1e-8, 0.0, scale, None) == 4
