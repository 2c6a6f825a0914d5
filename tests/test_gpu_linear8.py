"""Products in 8 bits against float64 of the same codes; the codes against their formula, to the bit.

Tolerance of a product: the output's rounding, u_T |y|, and fp32 sums.  Products of two codes are exact in fp32; a block of 128 columns is added up
in some order (at most 128 roundings of 2^-23 of the sum of magnitudes: the tensor core cuts off, it does not round), and the blocks' sums, with
two roundings for their scales, after one another: (128 + 3 + blocks) 2^-23 sum |x| |w|.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _formula(x, weight):
    """Codes and scales in elementary operations."""
    n, k = x.shape
    rb = 128 if weight else 1
    nb, kb = -(-n // rb), -(-k // 128)
    a = torch.zeros(nb * rb, kb * 128, device=x.device)
    a[:n, :k] = x.float()
    a = a.view(nb, rb, kb, 128)
    largest = a.abs().amax((1, 3), keepdim=True)
    largest = torch.where(largest < 2.0 ** -100, 0.0, largest)
    codes = (a * torch.where(largest > 0, largest.reciprocal() * 448, 0.0)).to(torch.float8_e4m3fn)
    return codes.view(nb * rb, -1)[:n, :k], (largest * (torch.ones((), device=DEV) / torch.full((), 448.0, device=DEV)))[:, 0, :, 0]


@pytest.mark.parametrize("rows,d", [(1, 1), (1, 128), (3, 100), (130, 257), (128, 512), (300, 2000), (77, 4096), (1000, 31)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_codes_follow_the_formula(rows, d, dtype):
    from addernetcuda_b200.linear8 import quantize_rows, quantize_weight
    torch.manual_seed(rows + d)
    x = (torch.randn(rows, d) * torch.exp(2 * torch.randn(d))).to(dtype).to(DEV)
    if rows > 2:
        x[1] = 0
        x[2] *= 1e-4
    for entry, weight in ((quantize_rows, False), (quantize_weight, True)):
        for t in (x, torch.cat([x, x], 1)[:, :d], torch.cat([x[:, :1], x], 1)[:, 1:]):
            got = entry(t)
            codes, scales = _formula(x, weight)
            assert torch.equal(got.scales, scales) and torch.equal(got.values.float(), codes.float())
            assert got.values.stride(0) % 16 == 0 or rows == 1
            assert torch.equal(got.dequantize(), (codes.float() * scales.repeat_interleave(128 if weight else 1, 0)[:rows].repeat_interleave(128, 1)[:, :d]))


def test_special_values():
    from addernetcuda_b200.linear8 import quantize_rows
    x = torch.randn(5, 256, device=DEV)
    x[0, 5] = float("nan")
    x[1, 130] = float("-inf")
    x[2] = 2.0 ** -101
    x[3] = 3e38
    v = quantize_rows(x).dequantize()
    assert v[0, :128].isnan().all() and torch.isfinite(v[0, 128:]).all() and v[1, 128:].isnan().all() and torch.isfinite(v[1, :128]).all()
    assert (v[2] == 0).all() and torch.allclose(v[3], x[3], rtol=1e-6) and torch.isfinite(v[4]).all()


def _case(m, k, n, dtype, seed=0, bias=False):
    from addernetcuda_b200.linear8 import quantize_rows, quantize_weight
    torch.manual_seed(seed)
    x = quantize_rows(torch.randn(m, k, device=DEV) * torch.exp(torch.randn(k, device=DEV)))
    w = quantize_weight(torch.randn(n, k, device=DEV))
    return x, w, torch.randn(n, device=DEV).to(dtype) if bias else None


def _near(y, x, w, bias):
    xd, wd = x.dequantize(torch.float32).double(), w.dequantize(torch.float32).double()
    # code * scale is rounded in dequantize: its own error, 2^-24 of each factor, is part of what is allowed
    want = xd.view(-1, xd.shape[-1]) @ wd.t()
    size = xd.view(-1, xd.shape[-1]).abs() @ wd.abs().t()
    blocks = -(-xd.shape[-1] // 128)
    if bias is not None:
        want = want + bias.double()
        size = size + bias.double().abs()
    want, size = want.view(y.shape), size.view(y.shape)
    off = (y.double() - want).abs()
    allowed = U[y.dtype] * want.abs() * (1 + 2.0 ** -8) + (131 + blocks + 2) * 2.0 ** -23 * size + (2.0 ** -25 if y.dtype == torch.float16 else 0.0)
    assert bool((off <= allowed).all()), f"off by {off.max():.3e}, worst ratio {(off / allowed).max():.3f} at {(off / allowed).argmax()}"


SIZES = [(1, 128, 128), (1, 1, 1), (1, 4096, 1000), (2, 100, 3), (7, 300, 129), (8, 512, 4096), (16, 128, 250), (17, 129, 127), (31, 1000, 640), (33, 256, 2000),
         (64, 2048, 513), (65, 384, 1024), (100, 130, 1001), (127, 640, 255), (128, 1024, 2048), (129, 96, 384), (200, 2000, 5003), (256, 512, 1536),
         (300, 4096, 500), (513, 250, 777), (1000, 1280, 3000), (1024, 512, 4096), (2050, 384, 1100), (2048, 64, 5000), (2000, 300, 2999), (60, 200, 1),
         (3, 100000, 70), (150, 1, 9000)]


@pytest.mark.parametrize("m,k,n", SIZES)
@pytest.mark.parametrize("dtype,bias", [(torch.float32, False), (torch.bfloat16, True), (torch.float16, False)])
def test_product(m, k, n, dtype, bias):
    from addernetcuda_b200.linear8 import linear_8bit
    x, w, b = _case(m, k, n, dtype, seed=m + k + n, bias=bias)
    if dtype == torch.float16:      # within fp16's range
        w = type(w)(w.values, w.scales / k)
    y = linear_8bit(x, w, b, dtype=dtype)
    assert y.dtype == dtype and y.shape == (m, n)
    _near(y, x, w, b)
    assert torch.equal(y, linear_8bit(x, w, b, dtype=dtype))      # always the same bits


@pytest.mark.parametrize("m,k,n", [(2970, 126, 11684), (1500, 64, 20484), (5000, 250, 8012), (3000, 100, 9996)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_short_tiles(m, k, n, dtype):
    """Several tiles a CTA, done faster than they are stored, the last ones of a row narrower than the others: nothing is stored from a buffer that the
    next tile writes."""
    from addernetcuda_b200.linear8 import linear_8bit
    x, w, _ = _case(m, k, n, dtype, seed=m)
    for _ in range(3):
        _near(linear_8bit(x, w, dtype=dtype), x, w, None)


def test_each_block_has_its_own_scale():
    """One code of 1 in each row: y is a product of two scales and a code, exactly."""
    from addernetcuda_b200.linear8 import Rows8, Weight8, linear_8bit
    torch.manual_seed(1)
    for m, k, n in ((5, 640, 300), (70, 640, 300), (300, 640, 700)):
        at = torch.randint(0, k, (m,), device=DEV)
        codes = torch.zeros(m, k, device=DEV)
        codes[torch.arange(m, device=DEV), at] = 1
        xs = 2.0 ** torch.randint(-8, 9, (m, 5), device=DEV).float()
        wv = torch.randint(-8, 9, (n, k), device=DEV).float()
        ws = 2.0 ** torch.randint(-8, 9, (-(-n // 128), 5), device=DEV).float()
        y = linear_8bit(Rows8(codes.to(torch.float8_e4m3fn), xs), Weight8(wv.to(torch.float8_e4m3fn), ws), dtype=torch.float32)
        want = wv[:, at].t() * xs.gather(1, at[:, None] // 128) * ws[torch.arange(n, device=DEV) // 128][:, at // 128].t()
        assert torch.equal(y, want)


def test_layouts():
    """Codes that are views, unaligned or of several axes; rows in 16 bits; nothing."""
    from addernetcuda_b200.linear8 import Rows8, Weight8, linear_8bit, quantize_rows
    x, w, _ = _case(12, 300, 200, torch.bfloat16)
    want = linear_8bit(x, w)
    assert want.dtype == torch.bfloat16
    dense = Rows8(x.values.contiguous(), x.scales), Weight8(w.values.contiguous(), w.scales)
    assert dense[0].values.stride(0) == 300
    assert torch.equal(linear_8bit(*dense), want)
    shifted = torch.empty(12, 400, dtype=torch.uint8, device=DEV)
    shifted[:, 5:305] = x.values.view(torch.uint8) if x.values.is_contiguous() else x.values.contiguous().view(torch.uint8)
    assert torch.equal(linear_8bit(Rows8(shifted.view(torch.float8_e4m3fn)[:, 5:305], x.scales), w), want)
    three = Rows8(x.values.contiguous().view(3, 4, 300), x.scales.view(3, 4, 3))
    assert torch.equal(linear_8bit(three, w), want.view(3, 4, 200))
    assert torch.equal(linear_8bit(Rows8(three.values[1, 2], three.scales[1, 2]), w), linear_8bit(Rows8(x.values[6:7], x.scales[6:7]), w)[0])
    strided = torch.empty(12, 6, device=DEV)[:, ::2].copy_(x.scales)
    assert torch.equal(linear_8bit(Rows8(x.values, strided), w), want)
    a = torch.randn(12, 300, device=DEV, dtype=torch.float16)
    y = linear_8bit(a, w)
    assert y.dtype == torch.float16 and torch.equal(y, linear_8bit(quantize_rows(a), w, dtype=torch.float16))
    assert linear_8bit(a[:0], w).shape == (0, 200)
    assert linear_8bit(x, Weight8(w.values[:0], w.scales[:0])).shape == (12, 0)


def test_what_lies_behind_the_rows_is_not_used():
    """Columns behind a row's last one, rows behind the last one: NaN codes there change nothing, and nothing is written there."""
    from addernetcuda_b200.linear8 import Rows8, Weight8, linear_8bit
    for m, k, n in ((3, 200, 130), (40, 200, 130), (140, 200, 130), (300, 1000, 300)):
        x, w, _ = _case(m, k, n, torch.float32)
        want = linear_8bit(x, w, dtype=torch.float32)

        def within(values):
            rows, cols = values.shape
            big = torch.full((rows + 130, cols // 16 * 16 + 64), 0x7F, dtype=torch.uint8, device=DEV)
            big[:rows, :cols] = values.contiguous().view(torch.uint8)
            return big.view(torch.float8_e4m3fn)[:rows, :cols]

        xs = torch.full((m + 200, x.scales.shape[1]), float("nan"), device=DEV)
        xs[:m] = x.scales
        assert torch.equal(linear_8bit(Rows8(within(x.values), xs[:m]), Weight8(within(w.values), w.scales), dtype=torch.float32), want)


def test_special_products():
    from addernetcuda_b200.linear8 import linear_8bit, quantize_rows, quantize_weight
    for m in (4, 40, 300):
        x = torch.randn(m, 256, device=DEV)
        x[1, 3] = float("nan")
        x[2] = 0
        w = torch.randn(140, 256, device=DEV)
        w[5, 200] = float("inf")      # its block stands for NaN: rows 0-127, columns 128-255
        y = linear_8bit(quantize_rows(x), quantize_weight(w), dtype=torch.float32)
        assert y[1].isnan().all() and y[:, :128].isnan().all() and (y[2, 128:] == 0).all() and torch.isfinite(y[3, 128:]).all()


def test_refusals():
    from addernetcuda_b200.linear8 import Linear8bit, Rows8, Weight8, linear_8bit, quantize_rows
    x, w, _ = _case(4, 128, 64, torch.float32)
    b = torch.zeros(64, device=DEV, dtype=torch.bfloat16)
    for bad, kind in ((lambda: linear_8bit(x, (w.values, w.scales)), TypeError), (lambda: linear_8bit(x, w, dtype=torch.float64), TypeError),
                      (lambda: linear_8bit(Rows8(x.values[:, :127], x.scales), w), ValueError), (lambda: linear_8bit(Rows8(x.values, x.scales[:3]), w), ValueError),
                      (lambda: linear_8bit(Rows8(x.values.float(), x.scales), w), TypeError), (lambda: linear_8bit(Rows8(x.values, x.scales.double()), w), TypeError),
                      (lambda: linear_8bit(x, Weight8(w.values, w.scales[:, :0])), ValueError), (lambda: linear_8bit(x, w, b[:63]), ValueError),
                      (lambda: linear_8bit(x, w, b.float()), ValueError), (lambda: linear_8bit(torch.randn(4, 128), w), RuntimeError),
                      (lambda: linear_8bit(torch.randn(4, 128, device=DEV, requires_grad=True), w), RuntimeError),
                      (lambda: linear_8bit(x, w, b.clone().requires_grad_()), RuntimeError), (lambda: quantize_rows(torch.zeros(4, 0, device=DEV)), ValueError),
                      (lambda: quantize_rows(torch.zeros(4, 4, device=DEV, dtype=torch.int32)), TypeError),
                      (lambda: Linear8bit(torch.nn.Conv2d(4, 4, 3).to(DEV)), ValueError), (lambda: Linear8bit(torch.nn.ReLU()), TypeError)):
        with pytest.raises(kind):
            bad()


def test_captured_on_another_stream_and_two_at_once():
    from addernetcuda_b200.linear8 import linear_8bit
    cases = [_case(m, k, n, torch.bfloat16, seed=i) for i, (m, k, n) in enumerate(((3, 4096, 2048), (70, 2048, 1024), (600, 512, 1000), (8, 8192, 256)))]
    want = [linear_8bit(x, w) for x, w, _ in cases]
    graphs = []
    for x, w, _ in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = linear_8bit(x, w)
        graphs.append((g, y))
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        for (g, y), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    eager = []
    for (x, w, _), s in zip(cases, streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            eager.append(linear_8bit(x, w))
    torch.cuda.synchronize()
    for (g, y), e, a in zip(graphs, eager, want):
        assert torch.equal(y, a) and torch.equal(e, a)


def test_offsets_beyond_32_bits():
    from addernetcuda_b200.linear8 import Rows8, Weight8, linear_8bit
    m, k, n = 70000, 128, 32000      # outputs
    x = Rows8(torch.ones(m, k, device=DEV).to(torch.float8_e4m3fn), torch.ones(m, 1, device=DEV))
    w = Weight8(torch.ones(n, k, device=DEV).to(torch.float8_e4m3fn), torch.ones(250, 1, device=DEV))
    x.values[-1] = 2
    y = linear_8bit(x, w)
    assert bool((y[-1] == 256).all()) and bool((y[-2] == 128).all()) and bool((y[::1000] == 128).all())
    del y, x, w
    m, k, n = 200, 8192, 270000      # weights
    w = Weight8(torch.empty(n, k, device=DEV, dtype=torch.float8_e4m3fn), torch.ones(-(-n // 128), 64, device=DEV))
    w.values.view(torch.uint8).fill_(0x38)      # 1.0
    w.values[-5:] = 2
    for rows in (3, 200):
        x = Rows8(torch.ones(rows, k, device=DEV).to(torch.float8_e4m3fn), torch.ones(rows, 64, device=DEV))
        y = linear_8bit(x, w)
        assert bool((y[:, -5:] == 2 * k).all()) and bool((y[:, :-5] == k).all())


def test_layers_of_networks():
    """quantize_linear: an nn.Linear, a 1x1 convolution and the head of this package's networks, near their own outputs."""
    from addernetcuda_b200 import resnet
    from addernetcuda_b200.inference import fold_batchnorm, quantize_linear
    from addernetcuda_b200.linear8 import Linear8bit
    torch.manual_seed(2)
    net = torch.nn.Sequential(torch.nn.Linear(100, 300), torch.nn.ReLU(), torch.nn.Linear(300, 17, bias=False)).to(DEV)
    x = torch.randn(50, 100, device=DEV)
    want = net(x).detach()
    quantize_linear(net)
    assert isinstance(net[0], Linear8bit) and isinstance(net[2], Linear8bit) and not net.training
    got = net(x)
    assert (got - want).norm() / want.norm() < 4 * 2.0 ** -4      # four roundings to e4m3, 2^-4 each at most
    again = torch.nn.Sequential(torch.nn.Linear(100, 300), torch.nn.ReLU(), torch.nn.Linear(300, 17, bias=False)).to(DEV)
    quantize_linear(again).load_state_dict(net.state_dict())
    assert torch.equal(again(x), got)
    for moved in (net.half(), net.cpu().cuda()):      # types of parameters; another device and back
        assert moved[0].values.dtype == torch.float8_e4m3fn and moved[0].scales.dtype == torch.float32 and moved[0].values.stride(0) == 112
        assert torch.equal(moved(x), got)
    assert net(x.half()).dtype == torch.float16
    tied = torch.nn.Linear(60, 60).to(DEV)
    both = quantize_linear(torch.nn.Sequential(tied, torch.nn.ReLU(), torch.nn.Sequential(tied)))
    assert isinstance(both[0], Linear8bit) and both[2][0] is both[0]
    assert isinstance(quantize_linear(tied), Linear8bit)
    conv = torch.nn.Conv2d(40, 24, 1).to(DEV)
    image = torch.randn(3, 40, 5, 7, device=DEV)
    y = Linear8bit(conv)(image)
    assert y.shape == (3, 24, 5, 7) and (y - conv(image)).norm() / conv(image).norm() < 2 * 2.0 ** -4
    cifar = resnet.resnet20().to(DEV)
    images = torch.randn(4, 3, 32, 32, device=DEV)
    seen = []
    with torch.no_grad():
        for m in cifar.modules():      # running statistics of these images: without them the untrained network's outputs are 0
            if isinstance(m, torch.nn.BatchNorm2d):
                m.momentum = 1.0
        cifar.train()(images)
        fold_batchnorm(cifar)
        # the layer's own output: the batch norm behind it divides by how far few images are apart
        cifar.fc.register_forward_hook(lambda module, args, out: seen.append(out))
        cifar(images)
        quantize_linear(cifar)
        cifar.fc.register_forward_hook(lambda module, args, out: seen.append(out))
        assert cifar(images).shape == (4, 10)
    want, got = seen
    assert isinstance(cifar.fc, Linear8bit) and got.shape == want.shape == (4, 10, 1, 1)
    assert (got - want).norm() / want.norm() < 2 * 2.0 ** -4
