"""RMS norm, the product in 8 bits, distillation and the verification of drafts as cases that can be timed and compared.

Four operators around the head of a network, each through its public entry point where `own` is true and in elementary torch operations
where it is not:

  rms     `rmsnorm.rms_norm`: y = h / sqrt(mean(h^2) + eps) * w over the last axis, with h = x + residual where there is a residual stream,
          and with `train` the gradients; with `eight` `rmsnorm.rms_norm_8bit`: y in e4m3 codes with a scale for each 128 columns of a row;
  mm8     `linear8.linear_8bit`: rows in e4m3 with a scale for each 128 columns (or, with `quantize`, in 16 or 32 bits and brought
          to that form within the call) times a weight in e4m3 with a scale for each 128 x 128;
  distill `distill.distillation`: the divergence of a network's classes from a teacher's best ones at a temperature, the log
          probability of a target class where there are targets, and with `train` the gradient of both with respect to the logits;
  verify  `drafts.verify_drafts`: how many of a sequence's drafted tokens stand against the target's probabilities, and the token that follows
          them, by given random numbers.

Codes are returned as tensors of float8_e4m3fn, with their scales.
"""
import math

import torch

own = False

DEV = "cuda:0"
EPS = 1e-6
IGNORE = -100
BLOCK = 128                 # columns (and rows of a weight) that share a scale
TOP = 448.0                 # the largest e4m3 value
TINY = 2.0 ** -100          # blocks whose largest value is below are zeros
_MAX_RMS, _MAX_LOGITS, _MAX_PROBS, _MAX_WEIGHT, _MAX_MM = 1 << 26, 1 << 28, 1 << 27, 1 << 27, 1 << 39
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    def rms(name, rows, width, dtype, wtype, residual, train, eight):
        return dict(name=name, op="rms", rows=rows, width=width, dtype=dtype, wtype=wtype, residual=residual, train=train, eight=eight)

    def mm8(name, tokens, inner, outer, dtype, quantize, bias):
        return dict(name=name, op="mm8", tokens=tokens, inner=inner, outer=outer, dtype=dtype, quantize=quantize, bias=bias)

    def distill(name, rows, classes, k, ragged, dtype, temperature, targets, train):
        return dict(name=name, op="distill", rows=rows, classes=classes, k=k, ragged=ragged, dtype=dtype, temperature=temperature,
                    targets=targets, train=train)

    def verify(name, sequences, drafts, classes, dtype, ragged, certain):
        return dict(name=name, op="verify", sequences=sequences, drafts=drafts, classes=classes, dtype=dtype, ragged=ragged, certain=certain)

    return [
        # one token in flight before a product in 8 bits: latency
        rms("rms_token_1x2048_bf16_8bit", 1, 2048, "bfloat16", "bfloat16", True, False, True),
        # a user's own width, odd in both extents, fp32 as the networks here train
        rms("rms_train_2051x1001_fp32", 2051, 1001, "float32", "float32", False, True, False),
        # a training batch of tokens, forward and backward, residual stream
        rms("rms_train_8192x4096_bf16", 8192, 4096, "bfloat16", "bfloat16", True, True, False),
        # a long prompt through a wide residual stream before a product in 8 bits
        rms("rms_prompt_8192x8192_bf16_8bit", 8192, 8192, "bfloat16", "float32", True, False, True),
        # the vocabulary's head for eight tokens in flight: the weight's bytes count
        mm8("mm8_head_8x4096x32000_bf16", 8, 4096, 32000, "bfloat16", False, False),
        # a layer of odd extents for part of a prompt, from activations in 16 bits
        mm8("mm8_chunk_333x2000x5003_bf16", 333, 2000, 5003, "bfloat16", True, True),
        # a wide layer for a long prompt: the tensor cores' rate counts
        mm8("mm8_prompt_8192x4096x16384_bf16", 8192, 4096, 16384, "bfloat16", False, False),
        # the head of the ImageNet network at its training batch, from a teacher's twenty best classes, with the labels
        distill("distill_train_256x1000_fp32_top20", 256, 1000, 20, False, "float32", 4.0, True, True),
        # how far a small model is from its teacher over given texts, an odd vocabulary
        distill("distill_score_2048x50257_bf16_top64", 2048, 50257, 64, True, "bfloat16", 1.0, False, False),
        # a training batch over a large vocabulary
        distill("distill_train_2048x128000_bf16_top32", 2048, 128000, 32, False, "bfloat16", 2.0, True, True),
        # one sequence, four drafted tokens: latency
        verify("verify_1x4x32000_fp32", 1, 4, 32000, "float32", False, False),
        # a full batch of a server over a large vocabulary, drafts of several lengths
        verify("verify_64x6x128000_bf16", 64, 6, 128000, "bfloat16", True, False),
    ]


# ------------------------------------------------------------------------------------------ drawn cases

def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    op = rng.choice(["rms", "mm8", "distill", "verify"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    if op == "rms":
        width = _log_int(rng, 24, 16384)
        width = width if rng.random() < 0.4 else -(-width // 8) * 8
        rows = _log_int(rng, 1, min(16384, _MAX_RMS // width))
        train = rng.random() < 0.5
        return dict(op=op, rows=rows, width=width, dtype=dtype, wtype=rng.choice([dtype, "float32"]), residual=rng.random() < 0.5,
                    train=train, eight=not train and rng.random() < 0.7)
    if op == "mm8":
        inner = _log_int(rng, 48, 8192)
        inner = inner if rng.random() < 0.4 else -(-inner // BLOCK) * BLOCK
        outer = _log_int(rng, 48, min(32768, _MAX_WEIGHT // inner))
        tokens = _log_int(rng, 1, min(8192, _MAX_MM // (inner * outer)))
        return dict(op=op, tokens=tokens, inner=inner, outer=outer, dtype=dtype, quantize=rng.random() < 0.4, bias=rng.random() < 0.4)
    if op == "distill":
        classes = _log_int(rng, 10, 200000)
        rows = _log_int(rng, 1, min(16384, _MAX_LOGITS // classes))
        return dict(op=op, rows=rows, classes=classes, k=min(_log_int(rng, 1, 64), classes // 2), ragged=rng.random() < 0.4, dtype=dtype,
                    temperature=rng.choice([1.0, 1.0, 2.0, 4.0, 0.7]), targets=rng.random() < 0.6, train=rng.random() < 0.6)
    classes, drafts = _log_int(rng, 10, 200000), rng.randint(1, 8)
    sequences = _log_int(rng, 1, min(256, _MAX_PROBS // (classes * (drafts + 1))))
    return dict(op=op, sequences=sequences, drafts=drafts, classes=classes, dtype=dtype, ragged=rng.random() < 0.5, certain=rng.random() < 0.25)


# ------------------------------------------------------------------------------------------ inputs

def _padded_rows(codes):
    """The same codes in a buffer whose rows begin at multiples of 16 bytes, as a loader lays them out once."""
    rows, n = codes.shape
    whole = torch.zeros(rows, -(-n // 16) * 16, dtype=torch.uint8, device=codes.device)
    whole[:, :n] = codes.view(torch.uint8)
    return whole.view(torch.float8_e4m3fn)[:, :n]


def _rows_in_8_bits(x):
    """e4m3 codes of rows in 32 bits, and a scale for each BLOCK columns."""
    rows, n = x.shape
    blocks = -(-n // BLOCK)
    a = torch.zeros(rows, blocks * BLOCK, device=x.device)
    a[:, :n] = x
    a = a.view(rows, blocks, BLOCK)
    largest = a.abs().amax(2, keepdim=True)
    largest = torch.where(largest < TINY, 0.0, largest)
    codes = (a * torch.where(largest > 0, TOP / largest, 0.0)).to(torch.float8_e4m3fn)
    return codes.view(rows, -1)[:, :n], (largest / TOP)[:, :, 0]


def _weight_in_8_bits(w):
    """The same of a weight, with a scale for each BLOCK x BLOCK."""
    n, k = w.shape
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    a = torch.zeros(nb * BLOCK, kb * BLOCK, device=w.device)
    a[:n, :k] = w
    a = a.view(nb, BLOCK, kb, BLOCK)
    largest = a.abs().amax((1, 3), keepdim=True)
    codes = (a * (TOP / largest)).to(torch.float8_e4m3fn)
    return codes.view(nb * BLOCK, -1)[:n, :k], (largest / TOP)[:, 0, :, 0].contiguous()


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device=DEV, generator=gen)

    def uniform(*shape):
        return torch.rand(*shape, device=DEV, generator=gen)

    dtype = TYPES[case["dtype"]]
    if case["op"] == "rms":
        shape = (case["rows"], case["width"])
        s = dict(case=case, x=(normal(*shape) * 1.5 + 0.3).to(dtype), w=(1 + 0.1 * normal(shape[1])).to(TYPES[case["wtype"]]))
        if case["residual"]:
            s["r"] = normal(*shape).to(dtype)
        if case["train"]:
            s["dy"] = normal(*shape).to(dtype)
            if case["residual"]:
                s["dh"] = normal(*shape).to(dtype)
            s["leaves"] = [s[k].requires_grad_() for k in ("x", "r", "w") if k in s]
        return s
    if case["op"] == "mm8":
        m, k, n = case["tokens"], case["inner"], case["outer"]
        # rows of a norm's output, some channels far larger than others
        x = normal(m, k) * torch.exp(0.7 * normal(k))
        w, ws = _weight_in_8_bits(normal(n, k) / math.sqrt(k))
        s = dict(case=case, w=_padded_rows(w), ws=ws, bias=(0.1 * normal(n)).to(dtype) if case["bias"] else None)
        if case["quantize"]:
            s["x"] = x.to(dtype)
        else:
            x, xs = _rows_in_8_bits(x)
            s["x"], s["xs"] = _padded_rows(x), xs.contiguous()
        return s
    if case["op"] == "distill":
        rows, classes, k = case["rows"], case["classes"], case["k"]
        logits = 2.5 * normal(rows, classes)
        targets = torch.randint(0, classes, (rows,), device=DEV, generator=gen)
        logits.scatter_add_(1, targets[:, None], torch.full((rows, 1), 6.0, device=DEV))
        # the teacher is surer of what the network half knows
        best, at = (1.3 * logits).topk(k, dim=1)
        s = dict(case=case, teacher=(best + normal(rows, k)).to(dtype), indices=at)
        if case["ragged"]:       # as many classes as make up most of the teacher's mass, which differs from row to row; some rows have none
            kept = torch.randint(0, k + 1, (rows, 1), device=DEV, generator=gen)
            s["indices"] = torch.where(torch.arange(k, device=DEV) < kept, at, -1)
        s["logits"] = logits.add_(normal(rows, classes)).to(dtype)
        if case["targets"]:
            skip = uniform(rows) < 0.05      # padding positions carry no target
            s["targets"] = torch.where(skip, IGNORE, targets)
        if case["train"]:
            s["logits"].requires_grad_()
            scale = (1024.0 if dtype == torch.float16 else 1.0) / rows         # a mean loss; fp16 trains with a loss scale
            s["g"] = scale * case["temperature"] ** 2 * uniform(rows)
            s["gl"] = -scale * uniform(rows) if case["targets"] else None
        return s
    b, k, classes = case["sequences"], case["drafts"], case["classes"]
    logits = 2.5 * normal(b, k + 1, classes)
    p = torch.softmax(logits, -1)
    drafter = torch.softmax(logits[:, :k] + normal(b, k, classes), -1)
    del logits
    tokens = torch.multinomial(drafter.view(b * k, classes), 1, generator=gen).view(b, k)
    if case["certain"]:          # a drafter that gives no probabilities: copied text
        keep = uniform(b, k) < 0.6
        tokens = torch.where(keep, p[:, :k].argmax(-1), tokens)
    s = dict(case=case, p=p.to(dtype), q=None if case["certain"] else drafter.to(dtype), tokens=tokens, u=uniform(b, k + 1), lengths=None)
    if case["ragged"]:
        s["lengths"] = torch.randint(0, k + 1, (b,), device=DEV, generator=gen)
    return s


# ------------------------------------------------------------------------------------------ plain forms

def _plain_rms(s):
    case = s["case"]
    with torch.no_grad():
        x, w = s["x"], s["w"].float()
        h = (x.float() + s["r"].float()).to(x.dtype) if case["residual"] else x
        hf = h.float()
        rs = 1.0 / torch.sqrt((hf * hf).mean(-1, keepdim=True) + EPS)
        xh = hf * rs
        out = {}
        if case["eight"]:
            out["values"], out["scales"] = _rows_in_8_bits(xh * w)
        else:
            out["y"] = (xh * w).to(x.dtype)
        if case["residual"]:
            out["h"] = h
        if case["train"]:
            dy = s["dy"].float()
            g = dy * w
            dx = rs * (g - xh * (g * xh).mean(-1, keepdim=True))
            if case["residual"]:
                dx = dx + s["dh"].float()
            out["dx"] = dx.to(x.dtype)
            if case["residual"]:
                out["dr"] = out["dx"]
            out["dw"] = (dy * xh).sum(0).to(s["w"].dtype)
        return out


def _spread(scales, rows, columns, block_rows):
    """Each scale at all the elements that share it."""
    if block_rows > 1:
        scales = scales.repeat_interleave(block_rows, 0)[:rows]
    return scales.repeat_interleave(BLOCK, 1)[:, :columns]


def _plain_mm8(s):
    case = s["case"]
    with torch.no_grad():
        m, k, n = case["tokens"], case["inner"], case["outer"]
        x, xs = _rows_in_8_bits(s["x"].float()) if case["quantize"] else (s["x"], s["xs"])
        y = (x.float() * _spread(xs, m, k, 1)) @ (s["w"].float() * _spread(s["ws"], n, k, BLOCK)).t()
        if case["bias"]:
            y = y + s["bias"].float()
        return dict(y=y.to(TYPES[case["dtype"]]))


def _plain_distill(s):
    case, tau = s["case"], s["case"]["temperature"]
    with torch.no_grad():
        zero = torch.zeros((), device=DEV)
        given = s["indices"] >= 0
        at = torch.where(given, s["indices"], 0)
        z = torch.where(given, s["teacher"].float() / tau, float("-inf"))
        z = z - torch.where(given.any(1, keepdim=True), z.amax(1, keepdim=True), zero)
        e = torch.exp(z)
        mass = e.sum(1, keepdim=True)
        t = torch.where(given, e / mass, zero)
        log_t = z - torch.log(mass)

        x = s["logits"].float()
        x = x - x.amax(1, keepdim=True)
        soft = x / tau
        e = torch.exp(soft)
        total = e.sum(1, keepdim=True)
        log_p = soft.gather(1, at) - torch.log(total)
        out = dict(divergence=torch.where(t > 0, t * (log_t - log_p), zero).sum(1))
        if case["train"]:
            g = s["g"][:, None] / tau
            grad = e / total * (g * t.sum(1, keepdim=True))
            grad.scatter_add_(1, at, -g * t)
        if case["targets"]:
            counts = s["targets"] != IGNORE
            target = torch.where(counts, s["targets"], 0)[:, None]
            e = torch.exp(x)
            total = e.sum(1, keepdim=True)
            out["log_prob"] = torch.where(counts, (x.gather(1, target) - torch.log(total))[:, 0], zero)
            if case["train"]:
                gl = torch.where(counts, s["gl"], zero)[:, None]
                grad -= e / total * gl
                grad.scatter_add_(1, target, gl)
        if case["train"]:
            out["grad"] = grad.to(s["logits"].dtype)
        return out


def _plain_verify(s):
    p, q, tokens, u = s["p"], s["q"], s["tokens"], s["u"].double()
    b, k, classes = *tokens.shape, p.shape[2]
    every = torch.arange(b, device=DEV)
    place = torch.arange(k + 1, device=DEV)
    lengths = torch.full((b,), k, device=DEV) if s["lengths"] is None else s["lengths"]
    one = torch.ones((), dtype=torch.float64, device=DEV)
    p_at = p[:, :k].gather(2, tokens[..., None])[..., 0].double()
    q_at = one if q is None else q.gather(2, tokens[..., None])[..., 0].double()
    stands = (u[:, :k] * q_at < p_at) & (place[:k] < lengths[:, None])
    n = stands.long().cumprod(1).sum(1)
    refused = (n < lengths)[:, None]
    last = n.clamp(max=k - 1)
    left = p[every, n].double()
    if q is None:
        gone = refused & (torch.arange(classes, device=DEV) == tokens[every, last][:, None])
        weight = torch.where(gone, 0.0, left)
    else:
        weight = (left - torch.where(refused, q[every, last].double(), 0.0)).clamp(min=0)
    weight = torch.where(weight.sum(1, keepdim=True) > 0, weight, left)
    reached = weight.cumsum(1)
    there = (reached > u[:, k:] * reached[:, -1:]) & (weight > 0)
    token = torch.where(there, torch.arange(classes, device=DEV), classes).amin(1)
    drafted = torch.cat([tokens, tokens[:, :1]], 1)
    out = torch.where(place < n[:, None], drafted, torch.where(place == n[:, None], token[:, None], -1))
    return dict(tokens=out, accepted=n)


# ------------------------------------------------------------------------------------------ the framework's calls

def _own_rms(s):
    from addernetcuda_b200.rmsnorm import rms_norm, rms_norm_8bit
    case = s["case"]
    x, w = s["x"], s["w"]
    if case["eight"]:
        if not case["residual"]:
            y = rms_norm_8bit(x, w, EPS)
            return dict(values=y.values, scales=y.scales)
        y, h = rms_norm_8bit(x, w, EPS, residual=s["r"])
        return dict(values=y.values, scales=y.scales, h=h)
    if not case["residual"]:
        y = rms_norm(x, (case["width"],), w, EPS)
        if not case["train"]:
            return dict(y=y)
        dx, dw = torch.autograd.grad(y, s["leaves"], s["dy"])
        return dict(y=y, dx=dx, dw=dw)
    y, h = rms_norm(x, (case["width"],), w, EPS, residual=s["r"])
    if not case["train"]:
        return dict(y=y, h=h)
    dx, dr, dw = torch.autograd.grad((y, h), s["leaves"], (s["dy"], s["dh"]))
    return dict(y=y, h=h, dx=dx, dr=dr, dw=dw)


def _own_mm8(s):
    from addernetcuda_b200.linear8 import Rows8, Weight8, linear_8bit
    case = s["case"]
    x = s["x"] if case["quantize"] else Rows8(s["x"], s["xs"])
    return dict(y=linear_8bit(x, Weight8(s["w"], s["ws"]), s["bias"], dtype=TYPES[case["dtype"]]))


def _own_distill(s):
    from addernetcuda_b200.distill import distillation
    case = s["case"]
    targets = s["targets"] if case["targets"] else None
    r = distillation(s["logits"], s["teacher"], s["indices"], temperature=case["temperature"], targets=targets, ignore_index=IGNORE)
    out = dict(divergence=r.divergence)
    if case["targets"]:
        out["log_prob"] = r.log_prob
    if case["train"]:
        if case["targets"]:
            out["grad"], = torch.autograd.grad([r.divergence, r.log_prob], s["logits"], [s["g"], s["gl"]])
        else:
            out["grad"], = torch.autograd.grad(r.divergence, s["logits"], s["g"])
    return out


def _own_verify(s):
    from addernetcuda_b200.drafts import verify_drafts
    r = verify_drafts(s["p"], s["q"], s["tokens"], s["u"], lengths=s["lengths"])
    return dict(tokens=r.tokens, accepted=r.accepted)


def run(state):
    op = state["case"]["op"]
    if own:
        return (_own_rms(state) if op == "rms" else _own_mm8(state) if op == "mm8" else _own_distill(state) if op == "distill"
                else _own_verify(state))
    return (_plain_rms(state) if op == "rms" else _plain_mm8(state) if op == "mm8" else _plain_distill(state) if op == "distill"
            else _plain_verify(state))


def work(case):
    size = torch.finfo(TYPES[case["dtype"]]).bits // 8
    if case["op"] == "rms":
        rows, d = case["rows"], case["width"]
        wide = torch.finfo(TYPES[case["wtype"]]).bits // 8
        read_and_written = 1 + 2 * case["residual"] + (not case["eight"]) + case["train"] * (2 + case["residual"])      # x; r, h; y; dy, dx; dh
        eight = rows * (d + 4 * -(-d // BLOCK)) if case["eight"] else 0
        return dict(bytes=read_and_written * rows * d * size + eight + (2 if case["train"] else 1) * d * wide,
                    flops=(15 if case["train"] else 8 if case["eight"] else 5) * rows * d)
    if case["op"] == "mm8":
        m, k, n = case["tokens"], case["inner"], case["outer"]
        kb = -(-k // BLOCK)
        x = m * k * size if case["quantize"] else m * (k + 4 * kb)
        return dict(bytes=x + n * k + 4 * kb * -(-n // BLOCK) + m * n * size + case["bias"] * n * size, flops=2 * m * k * n)
    if case["op"] == "distill":
        rows, n, k = case["rows"], case["rows"] * case["classes"], case["k"]
        per_row = k * (size + 8) + 4 + 12 * case["targets"] + case["train"] * (4 + 4 * case["targets"])
        return dict(bytes=n * size * (2 if case["train"] else 1) + rows * per_row, flops=(5 + 5 * case["targets"]) * (2 if case["train"] else 1) * n)
    # one row of the target's probabilities for each sequence, and one of the drafter's where a token is refused; single values of the others
    b, k, classes = case["sequences"], case["drafts"], case["classes"]
    rows = 1 if case["certain"] else 2
    return dict(bytes=b * (rows * (classes + k) * size + k * 8 + (k + 1) * 12 + 8), flops=5 * b * classes)


# ------------------------------------------------------------------------------------------ 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rms":
        out = {}
        with torch.no_grad():
            x, w = s["x"].double(), s["w"].double()
            if case["residual"]:       # the stream is held in its own type, and the norm is taken of what is held
                out["h"] = (x + s["r"].double()).to(s["x"].dtype).double()
                x = out["h"]
            z = x * torch.rsqrt(x.square().sum(-1, keepdim=True) / case["width"] + EPS)
            if case["eight"]:          # codes are decided by arithmetic in 32 bits; their scales have a value in 64
                parts = torch.split((z * w).abs(), BLOCK, dim=1)
                out["values"], out["scales"] = None, torch.stack([a.max(1).values for a in parts], 1) / TOP
            else:
                out["y"] = z * w
            if case["train"]:
                dy = s["dy"].double()
                a = dy * w
                root = torch.rsqrt(x.square().sum(-1, keepdim=True) / case["width"] + EPS)
                dx = a * root - x * root ** 3 * (a * x).sum(-1, keepdim=True) / case["width"]
                out["dx"] = dx + s["dh"].double() if case["residual"] else dx
                if case["residual"]:
                    out["dr"] = out["dx"]
                out["dw"] = torch.einsum("ij,ij->j", dy, z)
        return out
    if case["op"] == "mm8":            # codes made within the call are decided by arithmetic in 32 bits: the product has a value of them
        m, k, n = case["tokens"], case["inner"], case["outer"]
        x, xs = _rows_in_8_bits(s["x"].float()) if case["quantize"] else (s["x"], s["xs"])
        y = torch.zeros(m, n, dtype=torch.float64, device=DEV)
        of_row = s["ws"].double()[torch.arange(n, device=DEV) // BLOCK]
        for b in range(-(-k // BLOCK)):
            part = slice(b * BLOCK, min(k, (b + 1) * BLOCK))
            y.addmm_(x[:, part].double() * xs[:, b:b + 1].double(), (s["w"][:, part].double() * of_row[:, b:b + 1]).t())
        return dict(y=y + s["bias"].double() if case["bias"] else y)
    if case["op"] == "distill":
        tau = case["temperature"]
        x = s["logits"].detach().double().requires_grad_(case["train"])
        given = s["indices"] >= 0
        log_t = torch.log_softmax((s["teacher"].double() / tau).masked_fill(~given, -1e300), 1)
        t = log_t.exp() * given
        log_p = (x / tau).gather(1, s["indices"].clamp(min=0)) - torch.logsumexp(x / tau, 1, keepdim=True)
        out = dict(divergence=(t * (log_t.masked_fill(~given, 0.0) - log_p)).sum(1))
        outputs, grads = [out["divergence"]], [s["g"].double()] if case["train"] else None
        if case["targets"]:
            counts = s["targets"] != IGNORE
            at_target = x.gather(1, s["targets"].clamp(min=0)[:, None])[:, 0] - torch.logsumexp(x, 1)
            out["log_prob"] = torch.where(counts, at_target, 0.0)
            outputs.append(out["log_prob"])
            if case["train"]:
                grads.append(s["gl"].double())
        if case["train"]:
            out["grad"], = torch.autograd.grad(outputs, x, grads)
        return {name: v.detach() for name, v in out.items()}
    return None      # the verification's answers are whole numbers, equal or not
