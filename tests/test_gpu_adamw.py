"""The AdamW step against float64, its 8-bit states bit by bit against the same arithmetic in plain torch operations.

Tolerances count roundings: m and v are two products and a sum, three roundings of 2^-24 relative to |b m| + |(1 - b) g|; the update has
some 16 fp32 operations, two of them approximate to 2^-22, so 32 roundings of 2^-24 relative to its size; p is rounded to its
type once (half a step, u |p|).
"""
import copy

import pytest
import torch

from tests.adamw_plain import decode, encode, moments, update64

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
HYPER = dict(lr=3e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.02)


def _near(name, got, want, limit):
    off = (got.double() - want).abs()
    assert bool((off <= limit).all()), f"{name}: off by {float(off.max()):.3e}, {float((off / limit.clamp(min=1e-300)).max()):.2f} of what is allowed"


def _make(sizes, dtype, seed=0, g_scale=1e-2):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    rnd = lambda n: torch.randn(n, device=DEV, generator=gen)      # noqa: E731
    p = [(0.1 * rnd(n)).to(dtype) for n in sizes]
    g = [(g_scale * rnd(n)).to(dtype) for n in sizes]
    m = [1e-3 * rnd(n) for n in sizes]
    v = [(1e-3 * rnd(n)).square() for n in sizes]
    steps = torch.zeros(len(sizes), 2, dtype=torch.int32, device=DEV)
    steps[:, 0] = torch.arange(len(sizes), device=DEV) % 7 * 13
    return p, g, m, v, steps


def _check_step(p, g, m, v, steps, before, hyper=HYPER, g_scale=1.0):
    """Compares tensors after a step with float64 from the copies before it."""
    b1, b2 = hyper["betas"]
    for i, (p0, m0, v0, t0) in enumerate(zip(*before)):
        gd = g[i].double() * g_scale
        m1 = b1 * m0.double() + (1 - b1) * gd
        v1 = b2 * v0.double() + (1 - b2) * gd * gd
        _near(f"m[{i}]", m[i], m1, 4 * 2.0 ** -24 * (b1 * m0.double().abs() + (1 - b1) * gd.abs()) + 1e-38)
        _near(f"v[{i}]", v[i], v1, 6 * 2.0 ** -24 * v1 + 1e-38)
        t = int(t0[0]) + 1
        p1 = update64(p0, m1, v1, t, hyper["lr"], b1, b2, hyper["eps"], hyper["weight_decay"])
        size = (hyper["lr"] / (1 - b1 ** t) * (b1 * m0.double().abs() + (1 - b1) * gd.abs()) / ((v1 / (1 - b2 ** t)).sqrt() + hyper["eps"]))
        _near(f"p[{i}]", p[i], p1, U[p[i].dtype] * p1.abs() * (1 + 2.0 ** -8) + 32 * 2.0 ** -24 * size + 4 * 2.0 ** -24 * p1.abs() +
              (2.0 ** -25 if p[i].dtype == torch.float16 else 0.0))
        assert steps[i].tolist() == [t, 0]


def _copies(*lists):
    return [[t.clone() for t in ts] for ts in lists]


SIZES = [1, 2, 3, 7, 8, 9, 255, 256, 257, 1000, 2047, 2048, 2049, 4096, 5000, 65536, 100003]


@pytest.mark.parametrize("dtype", list(U), ids=str)
def test_states_in_32_bits(dtype):
    from addernetcuda_b200.optim import adamw_step
    p, g, m, v, steps = _make(SIZES, dtype)
    for _ in range(3):
        before = _copies(p, m, v, list(steps))
        adamw_step(p, g, m, v, steps, **HYPER)
        _check_step(p, g, m, v, steps, before)


@pytest.mark.parametrize("count", [47, 48, 49, 480, 481, 1100])
def test_any_number_of_tensors(count):
    """Tables of 48 and 480 tensors, and several launches."""
    from addernetcuda_b200.optim import adamw_step
    sizes = [(i * 37) % 301 + 1 for i in range(count)]
    sizes[count // 2] = 9000
    p, g, m, v, steps = _make(sizes, torch.float32)
    before = _copies(p, m, v, list(steps))
    adamw_step(p, g, m, v, list(steps), **HYPER)      # steps as a list, too
    _check_step(p, g, m, v, steps, before)


def _eight(sizes, dtype, seed=0, g_scale=1e-2):
    from addernetcuda_b200.optim import scale_count
    p, g, m, v, steps = _make(sizes, dtype, seed, g_scale)
    m, sm = map(list, zip(*(encode(t, True) for t in m)))
    v, sv = map(list, zip(*(encode(t, False) for t in v)))
    assert all(s.numel() == scale_count(t.numel()) for s, t in zip(sm, m))
    return p, g, m, v, sm, sv, steps


@pytest.mark.parametrize("dtype", list(U), ids=str)
def test_states_in_8_bits_bit_by_bit(dtype):
    from addernetcuda_b200.optim import adamw_state_values, adamw_step
    p, g, m, v, sm, sv, steps = _eight(SIZES, dtype)
    b1, b2 = HYPER["betas"]
    for _ in range(3):
        before = _copies(p, m, v, sm, sv, list(steps))
        adamw_step(p, g, m, v, steps, exp_avg_scales=sm, exp_avg_sq_scales=sv, **HYPER)
        for i in range(len(p)):
            p0, m0, v0, sm0, sv0, t0 = (b[i] for b in before)
            m1, v1 = moments(g[i].float(), decode(m0, sm0, True), decode(v0, sv0, False), b1, b2)
            for codes, scales, x, signed in ((m[i], sm[i], m1, True), (v[i], sv[i], v1, False)):
                want, want_scales = encode(x, signed)
                assert torch.equal(codes, want) and torch.equal(scales, want_scales), i
                assert torch.equal(adamw_state_values(codes, scales, signed), decode(codes, scales, signed))
            t = int(t0[0]) + 1
            p1 = update64(p0, m1, v1, t, HYPER["lr"], b1, b2, HYPER["eps"], HYPER["weight_decay"])
            size = HYPER["lr"] / (1 - b1 ** t) * m1.double().abs() / ((v1.double() / (1 - b2 ** t)).sqrt() + HYPER["eps"])
            _near(f"p[{i}]", p[i], p1, U[dtype] * p1.abs() * (1 + 2.0 ** -8) + 32 * 2.0 ** -24 * size + 4 * 2.0 ** -24 * p1.abs() +
                  (2.0 ** -25 if dtype == torch.float16 else 0.0))
            assert steps[i].tolist() == [t, 0]


def test_8_bit_blocks_of_zeros_tiny_and_mixed_values():
    from addernetcuda_b200.optim import adamw_step
    n = 256 * 6
    g = torch.zeros(n, device=DEV)
    g[256:512] = 1e-25                                              # v below what a block holds: stored as zeros
    g[512:768] = 10.0 ** torch.linspace(-18, 3, 256, device=DEV)    # most of the block far below its largest value
    g[768:1024] = -torch.rand(256, device=DEV)
    g[1024] = float("inf")
    g[1280] = float("nan")
    p, m, v = torch.ones(n, device=DEV), torch.zeros(n, dtype=torch.uint8, device=DEV), torch.zeros(n, dtype=torch.uint8, device=DEV)
    sm, sv = torch.zeros(6, device=DEV), torch.zeros(6, device=DEV)
    steps = torch.zeros(1, 2, dtype=torch.int32, device=DEV)
    adamw_step([p], [g], [m], [v], steps, exp_avg_scales=[sm], exp_avg_sq_scales=[sv], lr=0.1, betas=(0.9, 0.99), weight_decay=0.0)
    m1, v1 = moments(g, torch.zeros(n, device=DEV), torch.zeros(n, device=DEV), 0.9, 0.99)
    for codes, scales, x, signed in ((m, sm, m1, True), (v, sv, v1, False)):
        want, want_scales = encode(x, signed)
        assert torch.equal(codes[:1024], want[:1024]) and torch.equal(scales[:4], want_scales[:4])
        assert not bool(decode(codes, scales, signed)[1024:].isfinite().any())      # a block with an infinity or a NaN has no values
    assert bool((p[:256] == 1.0).all()) and bool(p[:1024].isfinite().all())
    assert float(sv[1]) == 0.0 and bool((v[256:512] == 0).all())
    assert bool((v[512:768][v1[512:768] > 0] >= 1).all()) and int((v[512:768] == 1).sum()) > 50


def test_alignment_and_shared_storage():
    """Views that start anywhere in one buffer, as gradient buckets hand them out; what lies beside them stays."""
    from addernetcuda_b200.optim import adamw_step
    for dtype in U:
        sizes = [5, 1, 300, 2048, 33, 4099]
        p, g, m, v, steps = _make(sizes, dtype)
        total = sum(sizes) + 1 + len(sizes)

        def scatter(ts):
            buf = torch.full((total,), 7.0, device=DEV).to(ts[0].dtype)
            out, at = [], 1
            for t in ts:
                buf[at:at + t.numel()] = t
                out.append(buf[at:at + t.numel()])
                at += t.numel() + 1
            return buf, out

        bufs, views = zip(*(scatter(ts) for ts in (p, g, m, v)))
        adamw_step(p, g, m, v, steps, **HYPER)
        steps2 = steps.clone()
        steps2[:, 0] -= 1
        adamw_step(*views, steps2, **HYPER)
        for ts, us in zip((p, g, m, v), views):
            assert all(torch.equal(a, b) for a, b in zip(ts, us))
        gaps, at = [0], 1
        for n in sizes:
            gaps.append(at + n)
            at += n + 1
        assert all(bool((b[gaps] == 7.0).all()) for b in bufs)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("bits", [32, 8])
def test_large_tensors(dtype, bits):
    """Several tiles a chunk, and tensors that end inside one."""
    from addernetcuda_b200.optim import adamw_step
    sizes = [20_000_003, 7, 65_537, 2_400_000]
    if bits == 32:
        p, g, m, v, steps = _make(sizes, dtype)
        before = _copies(p, m, v, list(steps))
        adamw_step(p, g, m, v, steps, **HYPER)
        _check_step(p, g, m, v, steps, before)
        return
    p, g, m, v, sm, sv, steps = _eight(sizes, dtype)
    before = _copies(p, m, v, sm, sv, list(steps))
    adamw_step(p, g, m, v, steps, exp_avg_scales=sm, exp_avg_sq_scales=sv, **HYPER)
    b1, b2 = HYPER["betas"]
    for i, (p0, m0, v0, sm0, sv0, t0) in enumerate(zip(*before)):
        m1, v1 = moments(g[i].float(), decode(m0, sm0, True), decode(v0, sv0, False), b1, b2)
        for codes, scales, x, signed in ((m[i], sm[i], m1, True), (v[i], sv[i], v1, False)):
            want, want_scales = encode(x, signed)
            assert torch.equal(codes, want) and torch.equal(scales, want_scales), i
        t = int(t0[0]) + 1
        p1 = update64(p0, m1, v1, t, HYPER["lr"], b1, b2, HYPER["eps"], HYPER["weight_decay"])
        size = HYPER["lr"] / (1 - b1 ** t) * m1.double().abs() / ((v1.double() / (1 - b2 ** t)).sqrt() + HYPER["eps"])
        _near(f"p[{i}]", p[i], p1, U[dtype] * p1.abs() * (1 + 2.0 ** -8) + 32 * 2.0 ** -24 * size + 4 * 2.0 ** -24 * p1.abs())
        assert steps[i].tolist() == [t, 0]


@pytest.mark.parametrize("dtype", list(U), ids=str)
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("first", [1, 2, 3, 4, 6])
def test_gradients_alone_at_other_addresses(dtype, bits, first):
    """All else is aligned, as when gradients are views of a bucket: the same bits as from an aligned gradient."""
    from addernetcuda_b200.optim import adamw_step
    make = _make if bits == 32 else _eight
    a, b = make(SIZES, dtype), make(SIZES, dtype)
    grads = []
    for g in b[1]:
        buf = torch.full((g.numel() + 16,), float("nan"), device=DEV).to(dtype)      # what lies beside a gradient is not used
        buf[first:first + g.numel()] = g
        grads.append(buf[first:first + g.numel()])
    for s, g in ((a, a[1]), (b, grads)):
        kw = dict(exp_avg_scales=s[4], exp_avg_sq_scales=s[5]) if bits == 8 else {}
        adamw_step(s[0], g, s[2], s[3], s[-1], **kw, **HYPER)
    for x, y in zip([a[0], *a[2:]], [b[0], *b[2:]]):
        assert all(torch.equal(t, u) for t, u in zip(list(x), list(y)))


def test_other_memory_orders_and_mixed_types():
    from addernetcuda_b200.optim import adamw_step
    torch.manual_seed(0)
    p0 = torch.randn(6, 5, 4, 3, device=DEV)
    g0 = torch.randn_like(p0)
    q0 = torch.randn(17, device=DEV)

    def state(t):
        return torch.zeros_like(t, dtype=torch.float32)

    a = [p0.clone(), q0.clone()]
    ga = [g0.clone(), torch.ones_like(q0)]
    sa = [state(t) for t in a], [state(t) for t in a], torch.zeros(2, 2, dtype=torch.int32, device=DEV)
    adamw_step(a, ga, *sa, **HYPER)
    b = [p0.to(memory_format=torch.channels_last), q0.clone()]
    sb = [state(t) for t in b], [state(t) for t in b], torch.zeros(2, 2, dtype=torch.int32, device=DEV)
    adamw_step(b, ga, *sb, **HYPER)           # the gradient lies in another order than its parameter
    assert all(torch.equal(x, y) for x, y in zip(a + sa[0] + sa[1], b + sb[0] + sb[1]))
    c = [p0.clone(), q0.bfloat16(), torch.randn(9, device=DEV).half(), q0.clone()]
    gc = [g0.clone(), torch.ones_like(c[1]), torch.ones_like(c[2]), torch.ones_like(q0)]
    sc = [state(t) for t in c], [state(t) for t in c], torch.zeros(4, 2, dtype=torch.int32, device=DEV)
    before = _copies(c, sc[0], sc[1], list(sc[2]))
    adamw_step(c, gc, *sc, **HYPER)
    _check_step(c, gc, *sc, before)
    assert torch.equal(c[0], a[0]) and torch.equal(c[3], a[1])


def test_device_values_of_lr_and_gradient_scale_and_betas_of_zero():
    from addernetcuda_b200.optim import adamw_step
    p, g, m, v, steps = _make([1000, 37], torch.float32)
    before = _copies(p, m, v, list(steps))
    adamw_step(p, g, m, v, steps, **{**HYPER, "lr": torch.tensor(HYPER["lr"], device=DEV)}, grad_scale=torch.tensor([0.25], device=DEV))
    _check_step(p, g, m, v, steps, before, g_scale=0.25)
    hyper = {**HYPER, "betas": (0.0, 0.0), "weight_decay": 0.0, "eps": 1e-6}
    before = _copies(p, m, v, list(steps))
    adamw_step(p, g, m, v, steps, **hyper)
    _check_step(p, g, m, v, steps, before, hyper)
    late = {**HYPER, "betas": (0.9, 0.999)}
    steps[:, 0] = 5_000_000
    before = _copies(p, m, v, list(steps))
    adamw_step(p, g, m, v, steps, **late)
    _check_step(p, g, m, v, steps, before, late)


def test_empty_tensors_and_shared_gradients():
    from addernetcuda_b200.optim import adamw_step
    p, g, m, v, steps = _make([4, 0, 4], torch.float32)
    g[2] = g[0]
    before = _copies(p, m, v, list(steps))
    adamw_step(p, g, m, v, steps, **HYPER)
    steps[1, 0] += 1
    _check_step(p, g, m, v, steps, before)


def test_refusals():
    from addernetcuda_b200.optim import adamw_state_values, adamw_step

    def attempt(error, match, **change):
        p, g, m, v, steps = _make([64, 64], torch.float32)
        args = dict(params=p, grads=g, exp_avgs=m, exp_avg_sqs=v, steps=steps)
        kw = dict(HYPER)
        for k, f in change.items():
            if k in args:
                args[k] = f(args)
            else:
                kw[k] = f(args)
        kept = [t.clone() for t in p]
        with pytest.raises(error, match=match):
            adamw_step(*args.values(), **kw)
        assert all(torch.equal(a, b) for a, b in zip(kept, p))      # nothing was done

    attempt(ValueError, "also those of another", params=lambda a: [a["params"][0]] * 2)
    attempt(ValueError, "also those of another", exp_avgs=lambda a: [a["exp_avgs"][0]] * 2)
    attempt(ValueError, "also those of another", exp_avg_sqs=lambda a: a["exp_avgs"])
    attempt(ValueError, "also those of another", steps=lambda a: [a["steps"][0]] * 2)
    attempt(ValueError, "gradient is also", grads=lambda a: a["params"])
    attempt(ValueError, "shape", grads=lambda a: [a["grads"][0], a["grads"][1][:32]])
    attempt(TypeError, "grads", grads=lambda a: [t.bfloat16() for t in a["grads"]])
    attempt(TypeError, "exp_avgs", exp_avgs=lambda a: [t.half() for t in a["exp_avgs"]])
    attempt(ValueError, "exp_avg_sqs", exp_avg_sqs=lambda a: [t[:60] for t in a["exp_avg_sqs"]])
    attempt(TypeError, "steps", steps=lambda a: a["steps"].float())
    attempt(ValueError, "steps", steps=lambda a: a["steps"][:1])
    attempt(ValueError, "steps", steps=lambda a: [t[:1] for t in a["steps"]])
    attempt(TypeError, "float32, bfloat16 or float16", params=lambda a: [t.double() for t in a["params"]])
    attempt(RuntimeError, "CUDA|devices", grads=lambda a: [t.cpu() for t in a["grads"]])
    attempt(ValueError, "fill its memory", params=lambda a: [torch.zeros(128, device=DEV)[::2], a["params"][1]])
    attempt(TypeError, "layout", grads=lambda a: [a["grads"][0].to_sparse(), a["grads"][1]])
    attempt(TypeError, "exp_avgs", exp_avg_scales=lambda a: [torch.zeros(1, device=DEV)] * 2, exp_avg_sq_scales=lambda a: [torch.zeros(1, device=DEV)] * 2)
    attempt(ValueError, "", betas=lambda a: (1.0, 0.9))
    attempt(TypeError, "lr", lr=lambda a: torch.tensor(1e-3, device=DEV, dtype=torch.float64))
    attempt(ValueError, "lr", lr=lambda a: torch.zeros(2, device=DEV))
    attempt(TypeError, "grad_scale", grad_scale=lambda a: 0.5)
    codes = torch.zeros(300, dtype=torch.uint8, device=DEV)
    with pytest.raises(ValueError, match="scales"):
        adamw_state_values(codes, torch.zeros(1, device=DEV), True)
    with pytest.raises(TypeError, match="codes"):
        adamw_state_values(codes.float(), torch.zeros(2, device=DEV), True)


def test_without_the_host_path_the_results_are_the_same(monkeypatch):
    from addernetcuda_b200 import _native
    from addernetcuda_b200.optim import adamw_step
    for make in (_make, _eight):
        a, b = make([1000, 3, 2048], torch.bfloat16), make([1000, 3, 2048], torch.bfloat16)
        for s in (a, b):
            with monkeypatch.context() as mp:
                if s is b:
                    mp.setattr(_native, "adamw", _native._absent)
                kw = dict(exp_avg_scales=s[4], exp_avg_sq_scales=s[5]) if len(s) == 7 else {}
                adamw_step(s[0], s[1], s[2], s[3], s[-1], **kw, **HYPER)
        for x, y in zip(a, b):
            assert all(torch.equal(t, u) for t, u in zip(list(x), list(y)))


def test_two_threads_at_once():
    """Each with tensors, lists and a stream of its own, emptied and filled again between the steps."""
    import threading

    from addernetcuda_b200.optim import adamw_step
    sets = [_make([1000, 3, 2048, 70000], torch.float32, seed=i) for i in range(2)]
    want = [_make([1000, 3, 2048, 70000], torch.float32, seed=i) for i in range(2)]
    for s in want:
        for _ in range(50):
            adamw_step(*s, **HYPER)
    torch.cuda.synchronize()
    failed = []

    def work(s):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(50):
                    lists = [list(ts) for ts in s[:4]]
                    adamw_step(*lists, s[4], **HYPER)
                    for ts in lists:
                        ts.clear()
                torch.cuda.current_stream().synchronize()
        except Exception as e:
            failed.append(e)

    threads = [threading.Thread(target=work, args=(s,)) for s in sets]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for s, w in zip(sets, want):
        assert all(torch.equal(a, b) for x, y in zip(s, w) for a, b in zip(list(x), list(y)))


def test_versions_tell_autograd_of_the_write():
    from addernetcuda_b200.optim import adamw_step
    p, g, m, v, steps = _make([8], torch.float32)
    w = p[0].requires_grad_()
    out = (w * w).sum()
    adamw_step([w], g, m, v, steps, **HYPER)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward()


# ------------------------------------------------------------------------------------------ the optimizer

def _params(dtype=torch.float32):
    torch.manual_seed(0)
    return [torch.nn.Parameter((0.1 * torch.randn(s, device=DEV)).to(dtype)) for s in ((64, 80), (80,), (3, 5, 3, 3), (1,), (8192,))]


def _grads(ps, seed):
    torch.manual_seed(seed)
    for p in ps:
        p.grad = (0.01 * torch.randn_like(p)).to(p.dtype)


def test_optimizer_against_torchs():
    from addernetcuda_b200.optim import AdamW
    a, b = _params(), [torch.nn.Parameter(p.detach().double()) for p in _params()]
    oa = AdamW([{"params": a[:2]}, {"params": a[2:], "weight_decay": 0.0, "lr": 1e-2}], **HYPER)
    ob = torch.optim.AdamW([{"params": b[:2]}, {"params": b[2:], "weight_decay": 0.0, "lr": 1e-2}], **HYPER)
    for i in range(6):
        _grads(a, i)
        for p, q in zip(a, b):
            q.grad = p.grad.double()
        if i == 3:
            a[1].grad = b[1].grad = None      # a parameter may miss a step: it counts its own
        oa.step()
        ob.step()
    for p, q in zip(a, b):
        # six updates of at most a learning rate (1e-2) each, 32 roundings each, and the rounding of p at each
        assert bool(((p.double() - q).abs() <= 6 * (32 * 2.0 ** -24 * 1e-2 * 3 + 2.0 ** -23 * q.abs())).all())
    assert [int(oa.state[p]["step"][0]) for p in a] == [6, 5, 6, 6, 6]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_goes_on_where_it_stopped(dtype, bits):
    from addernetcuda_b200.optim import AdamW
    a = _params(dtype)
    oa = AdamW(a, state_bits=bits, **HYPER)
    for i in range(2):
        _grads(a, i)
        oa.step()
    assert ("exp_avg_scale" in oa.state[a[0]]) == (bits == 8) and "exp_avg_scale" not in oa.state[a[1]]      # small ones keep 32 bits
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    ob = AdamW(b, state_bits=bits)
    ob.load_state_dict(copy.deepcopy(oa.state_dict()))
    for i in range(2, 4):
        for ps, o in ((a, oa), (b, ob)):
            _grads(ps, i)
            o.step()
    for p, q in zip(a, b):
        assert torch.equal(p, q)
        assert oa.state[p].keys() == ob.state[q].keys()
        assert all(torch.equal(oa.state[p][k], ob.state[q][k]) and oa.state[p][k].dtype == ob.state[q][k].dtype for k in oa.state[p])


def test_captured_steps_count_and_follow_the_learning_rate():
    from addernetcuda_b200.optim import AdamW
    for bits in (32, 8):
        a, b = _params(), _params()
        lr = torch.tensor(1e-3, device=DEV)
        oa, ob = AdamW(a, lr=lr, state_bits=bits), AdamW(b, lr=1e-3, state_bits=bits)
        with pytest.raises(RuntimeError, match="cannot be captured"):
            _grads(a, 0)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                oa.step()
        side = torch.cuda.Stream()
        _grads(a, 0)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            oa.step()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            oa.step()
        for i, rate in ((0, 1e-3), (1, 1e-3), (2, 5e-4), (3, 2e-4)):
            if i:
                lr.fill_(rate)
                torch.manual_seed(i)
                for p in a:
                    p.grad.copy_(0.01 * torch.randn_like(p))
                g.replay()
            _grads(b, i)
            ob.param_groups[0]["lr"] = rate
            ob.step()
        assert all(torch.equal(p, q) for p, q in zip(a, b)), bits


def test_closure_and_missing_gradients():
    from addernetcuda_b200.optim import AdamW
    ps = _params()
    opt = AdamW(ps)
    kept = [p.detach().clone() for p in ps]
    opt.step()      # no gradients: nothing happens
    assert all(torch.equal(p, q) for p, q in zip(ps, kept))

    def closure():
        opt.zero_grad()
        loss = sum((p * p).sum() for p in ps)
        loss.backward()
        return loss

    first = opt.step(closure)
    assert float(opt.step(closure)) < float(first)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("eps", [0.0, 1e-30])
def test_second_moments_below_the_normal_range(dtype, eps):
    """Gradients of 1e-20 to 1e-18 leave second moments of 2^-138 to 2^-124: the update by their root is as large as any other."""
    from addernetcuda_b200.optim import adamw_step
    b1, b2 = HYPER["betas"]
    hyper = {**HYPER, "eps": eps, "weight_decay": 0.0}
    gen = torch.Generator(device=DEV)
    gen.manual_seed(3)
    sizes = [5, 2048, 2051, 5000]
    rnd = lambda n: torch.rand(n, device=DEV, generator=gen)      # noqa: E731
    p = [(rnd(n) + 0.5).to(dtype) for n in sizes]
    g = [(10.0 ** (-20 + 2 * rnd(n)) * (1 - 2 * (rnd(n) < 0.5).float())).to(dtype) for n in sizes]
    m, v = ([torch.zeros(n, device=DEV) for n in sizes] for _ in range(2))
    steps = torch.zeros(len(sizes), 2, dtype=torch.int32, device=DEV)
    for t in (1, 2, 3):
        before = _copies(p, m, v)
        adamw_step(p, g, m, v, steps, **hyper)
        for i, (p0, m0, v0) in enumerate(zip(*before)):
            m1, v1 = moments(g[i].float(), m0, v0, b1, b2)
            assert torch.equal(m[i], m1) and torch.equal(v[i], v1) and bool((v1 > 0).all())
            p1 = update64(p0, m1, v1, t, hyper["lr"], b1, b2, eps, 0.0)
            size = hyper["lr"] / (1 - b1 ** t) * m1.double().abs() / ((v1.double() / (1 - b2 ** t)).sqrt() + eps)
            assert float(size.max()) > 0.5 * hyper["lr"]
            _near(f"p[{i}]", p[i], p1, U[dtype] * p1.abs() * (1 + 2.0 ** -8) + 32 * 2.0 ** -24 * size + 4 * 2.0 ** -24 * p1.abs())
    for a in m + g:      # a first moment of 0 moves nothing
        a.zero_()
    before = _copies(p)
    adamw_step(p, g, m, v, steps, **hyper)
    assert all(torch.equal(a, b) for a, b in zip(p, before[0]))


def test_second_moments_below_the_normal_range_before_8_bit_states_are_stored():
    """The update uses v as it is before it is stored.  8-bit steps have two kernels by eps: both sides of the rule."""
    from addernetcuda_b200.optim import adamw_step
    n, (b1, b2) = 256 * 9 + 5, HYPER["betas"]
    gen = torch.Generator(device=DEV)
    gen.manual_seed(4)
    border = 2.0 ** -39 / (1 - b2) ** 0.5
    for exponent, eps in ((-20, 0.0), (-20, 1e-30), (-12, 0.99 * border), (-12, border * (1 + 1e-6)), (-20, border * (1 + 1e-6))):
        g = 10.0 ** (exponent + 2 * torch.rand(n, device=DEV, generator=gen))
        p, m, v = torch.ones(n, device=DEV), torch.zeros(n, dtype=torch.uint8, device=DEV), torch.zeros(n, dtype=torch.uint8, device=DEV)
        sm, sv, steps = torch.zeros(10, device=DEV), torch.zeros(10, device=DEV), torch.zeros(1, 2, dtype=torch.int32, device=DEV)
        adamw_step([p], [g], [m], [v], steps, exp_avg_scales=[sm], exp_avg_sq_scales=[sv], **{**HYPER, "eps": eps, "weight_decay": 0.0})
        m1, v1 = moments(g, torch.zeros(n, device=DEV), torch.zeros(n, device=DEV), b1, b2)
        p1 = update64(torch.ones(n, device=DEV), m1, v1, 1, HYPER["lr"], b1, b2, eps, 0.0)
        size = HYPER["lr"] / (1 - b1) * m1.double() / ((v1.double() / (1 - b2)).sqrt() + eps)
        _near(f"p, eps {eps}", p, p1, (1 + 4) * 2.0 ** -24 * p1.abs() + 32 * 2.0 ** -24 * size)


def test_lazily_negated_gradients():
    from addernetcuda_b200.optim import adamw_step
    negated = lambda v: torch.complex(torch.zeros_like(v), v).conj().imag      # noqa: E731
    p, g, m, v, steps = _make([1, 1, 40], torch.float32)
    before = _copies(p, m, v, list(steps))
    lazy = [negated(t) for t in g]
    assert all(t.is_neg() for t in lazy) and lazy[0].is_contiguous()
    adamw_step(p, lazy, m, v, steps, **HYPER)
    _check_step(p, [-t for t in g], m, v, steps, before)
    with pytest.raises(ValueError, match="lazily negated"):
        adamw_step([lazy[0]], [g[0]], m[:1], v[:1], steps[:1], **HYPER)
    with pytest.raises(ValueError, match="lazily negated"):
        adamw_step(p[:1], g[:1], [negated(m[0])], v[:1], steps[:1], **HYPER)
