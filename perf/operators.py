"""Layer norm, log probabilities and the AdamW step as cases that can be timed and compared.

Three operators around a network whose last axis holds features or classes, each through its public entry point where
`own` is true and in elementary torch operations where it is not:

  ln      `layernorm.layer_norm`: y = (h - mean) / sqrt(var + eps) * w + b over the last axis, with h = x + residual where there is a
          residual stream, and with `train` the gradients;
  lp      `logprobs.token_log_probs`: log probability of the target class of each row, entropy of the row, the k most probable classes
          (ties: lowest index), and with `train` the gradient of all of them with respect to the logits;
  adamw   `optim.adamw_step`: one AdamW step over all tensors of a model, states in 32 bits or as 8-bit codes with a scale for each
          256 values.

Tensors of one model lie in one buffer at multiples of 256 elements (an allocator's or a bucket's layout); what lies between them is
zero and stays zero, so that the plain form may work on the buffer as a whole.
"""
import math

import torch

own = False

DEV = "cuda:0"
EPS = 1e-5
IGNORE = -100
BLOCK = 256                 # values that share a scale; tensors of a model start at multiples of it
TOP_M, TOP_V = 248.0, 63488.0     # largest magnitudes of the codes: (1 + 15/16) 2^7 and (1 + 15/16) 2^15
TINY = 2.0 ** -100          # blocks whose largest value is below are stored as zeros
ADAMW = dict(lr=1e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.01)
_MAX_LN, _MAX_LP, _MAX_ADAMW = 1 << 26, 1 << 28, 200_000_000       # elements of drawn cases
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    def ln(name, rows, width, dtype, wtype, residual, train):
        return dict(name=name, op="ln", rows=rows, width=width, dtype=dtype, wtype=wtype, residual=residual, train=train)

    def lp(name, rows, classes, pad, dtype, top_k, entropy, masked, train):
        return dict(name=name, op="lp", rows=rows, classes=classes, pad=pad, dtype=dtype, top_k=top_k, entropy=entropy, masked=masked,
                    train=train)

    def adamw(name, net, width, layers, dtype, bits):
        return dict(name=name, op="adamw", net=net, width=width, layers=layers, dtype=dtype, bits=bits)

    return [
        # one token in flight through a residual stream: latency
        ln("ln_token_1x2048_bf16", 1, 2048, "bfloat16", "bfloat16", True, False),
        # a training batch of tokens, forward and backward, residual stream
        ln("ln_train_8192x4096_bf16", 8192, 4096, "bfloat16", "bfloat16", True, True),
        # a user's own width, odd in both extents, fp32 as the networks here train
        ln("ln_train_2051x1001_fp32", 2051, 1001, "float32", "float32", False, True),
        # activation planes of a 256-channel 14x14 stage, each image normalised as a whole
        ln("ln_train_64x50176_fp32", 64, 50176, "float32", "float32", False, True),
        # sampling: a few sequences, a padded vocabulary, masked classes, the 20 best alternatives
        lp("lp_sample_4x32000_bf16_top20", 4, 32000, 64, "bfloat16", 20, True, True, False),
        # the head of the ImageNet network at its training batch: loss, its gradient
        lp("lp_train_256x1000_fp32", 256, 1000, 0, "float32", 0, False, False, True),
        # scoring given texts: an odd vocabulary, five alternatives and the entropy at each position
        lp("lp_score_4096x50257_bf16_top5", 4096, 50257, 0, "bfloat16", 5, True, False, False),
        # a training batch over a large vocabulary, with an entropy term
        lp("lp_train_2048x128000_bf16", 2048, 128000, 0, "bfloat16", 0, True, False, True),
        # the CIFAR network: 66 small tensors, where launches and host time count
        adamw("adamw_resnet20_fp32", "resnet20", 0, 0, "float32", 32),
        # the ImageNet network: 163 tensors from 64 to 2.4 million elements
        adamw("adamw_resnet50_fp32", "resnet50", 0, 0, "float32", 32),
        # blocks of a token model of odd width, states in 32 bits beside bf16 weights
        adamw("adamw_blocks_1001x4_bf16", "blocks", 1001, 4, "bfloat16", 32),
        # the largest: states in 8 bits, read out afterwards as a checkpoint does
        adamw("adamw_blocks_2048x4_bf16_8bit", "blocks", 2048, 4, "bfloat16", 8),
    ]


# ------------------------------------------------------------------------------------------ drawn cases

def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["ln", "lp", "adamw"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    if op == "ln":
        width = _log_int(rng, 24, 60000)
        width = width if rng.random() < 0.4 else -(-width // 8) * 8
        rows = _log_int(rng, 1, min(16384, _MAX_LN // width))
        return dict(op=op, rows=rows, width=width, dtype=dtype, wtype=rng.choice([dtype, "float32"]), residual=rng.random() < 0.5,
                    train=rng.random() < 0.6)
    if op == "lp":
        classes = _log_int(rng, 10, 200000)
        top_k = rng.choice([0, 0, 1, 5, 20])
        rows = _log_int(rng, 1, min(16384, (_MAX_LP >> (1 if top_k else 0)) // classes))
        train = rng.random() < 0.5
        return dict(op=op, rows=rows, classes=classes, pad=rng.choice([0, 0, rng.randrange(1, 64)]), dtype=dtype,
                    top_k=min(top_k, classes // 2), entropy=rng.random() < 0.6, masked=not train and rng.random() < 0.3, train=train)
    width = _log_int(rng, 24, 2048)
    layers = _log_int(rng, 1, 24)
    layers = max(1, min(layers, _MAX_ADAMW // (12 * width * width)))
    return dict(op=op, net="blocks", width=width, layers=layers, dtype=dtype, bits=rng.choice([32, 8]))


# ------------------------------------------------------------------------------------------ inputs

def _sizes(case):
    """Elements of each tensor of a model."""
    if case["net"] == "blocks":
        w = case["width"]
        return [w * w, w * w, w * w, w * w, 4 * w * w, 4 * w, 4 * w * w, w, w] * case["layers"]
    if case["net"] == "resnet20":
        sizes, ci = [3 * 16 * 9, 16, 16], 16
        for stage, co in enumerate((16, 32, 64)):
            for block in range(3):
                sizes += [ci * co * 9, co, co, co * co * 9, co, co] + ([ci * co, co, co] if stage and block == 0 else [])
                ci = co
        return sizes + [64 * 10, 10, 10]
    sizes, ci = [3 * 64 * 49, 64, 64], 64
    for c, blocks in ((64, 3), (128, 4), (256, 6), (512, 3)):
        for block in range(blocks):
            sizes += [ci * c, c, c, c * c * 9, c, c, c * 4 * c, 4 * c, 4 * c] + ([ci * 4 * c, 4 * c, 4 * c] if block == 0 else [])
            ci = 4 * c
    return sizes + [2048 * 1000, 1000, 1000, 1000]


def _padded(n):
    return -(-n // BLOCK) * BLOCK


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device=DEV, generator=gen)

    dtype = TYPES[case["dtype"]]
    if case["op"] == "ln":
        shape = (case["rows"], case["width"])
        wtype = TYPES[case["wtype"]]
        s = dict(case=case, x=(normal(*shape) * 1.5 + 0.3).to(dtype), w=(1 + 0.1 * normal(shape[1])).to(wtype),
                 b=(0.1 * normal(shape[1])).to(wtype))
        if case["residual"]:
            s["r"] = normal(*shape).to(dtype)
        if case["train"]:
            s["dy"] = normal(*shape).to(dtype)
            if case["residual"]:
                s["dh"] = normal(*shape).to(dtype)
            s["leaves"] = [s[k].requires_grad_() for k in ("x", "r", "w", "b") if k in s]
        return s
    if case["op"] == "lp":
        rows, classes = case["rows"], case["classes"]
        targets = torch.randint(0, classes, (rows,), device=DEV, generator=gen)
        logits = 2.5 * normal(rows, classes + case["pad"])
        logits.scatter_add_(1, targets[:, None], torch.full((rows, 1), 5.0, device=DEV))
        if case["masked"]:       # a constrained vocabulary: three classes in ten are out
            out = torch.rand(logits.shape, device=DEV, generator=gen) < 0.3
            out.scatter_(1, targets[:, None], False)
            logits.masked_fill_(out, float("-inf"))
        s = dict(case=case, logits=logits.to(dtype)[:, :classes], targets=targets)
        if case["train"]:
            skip = torch.rand(rows, device=DEV, generator=gen) < 0.05      # padding positions carry no target
            s["targets"] = torch.where(skip, IGNORE, targets)
            s["logits"].requires_grad_()
            scale = (1024.0 if dtype == torch.float16 else 1.0) / rows         # a mean loss; fp16 trains with a loss scale
            s["g"] = -scale * torch.rand(rows, device=DEV, generator=gen)
            s["ge"] = 0.01 * scale * normal(rows) if case["entropy"] else None
            s["gt"] = 0.1 * scale * normal(rows, case["top_k"]) if case["top_k"] else None
        return s
    sizes = _sizes(case)
    starts, total = [], 0
    for n in sizes:
        starts.append(total)
        total += _padded(n)
    inside = torch.zeros(total, dtype=torch.bool, device=DEV)
    for a, n in zip(starts, sizes):
        inside[a:a + n] = True
    g = (1e-3 * normal(total) * inside).to(dtype)
    m = 3e-4 * normal(total) * inside
    v = (1e-3 * normal(total) * inside) ** 2 * 0.3 + 1e-8 * inside
    s = dict(case=case, flat_p=(0.02 * normal(total) * inside).to(dtype), flat_g=g)
    if case["bits"] == 32:
        s["flat_m"], s["flat_v"] = m, v
    else:
        s["flat_m"], s["scale_m"] = _encode(m, True)
        s["flat_v"], s["scale_v"] = _encode(v, False)
    for k in ("p", "g", "m", "v"):
        s[k] = [s["flat_" + k][a:a + n] for a, n in zip(starts, sizes)]
    if case["bits"] == 8:
        for k in ("m", "v"):
            s["s" + k] = [s["scale_" + k][a // BLOCK:(a + _padded(n)) // BLOCK] for a, n in zip(starts, sizes)]
    s["steps"] = torch.zeros(len(sizes), 2, dtype=torch.int32, device=DEV)      # steps taken, and a word of the kernel's
    s["steps"][:, 0] = 1000
    return s


# ------------------------------------------------------------------------------------------ plain forms

def _plain_ln(s):
    case = s["case"]
    with torch.no_grad():
        x, w = s["x"], s["w"].float()
        h = (x.float() + s["r"].float()).to(x.dtype) if case["residual"] else x
        hf = h.float()
        c = hf - hf.mean(-1, keepdim=True)
        rs = 1.0 / torch.sqrt((c * c).mean(-1, keepdim=True) + EPS)
        xh = c * rs
        out = dict(y=(xh * w + s["b"].float()).to(x.dtype))
        if case["residual"]:
            out["h"] = h
        if case["train"]:
            dy = s["dy"].float()
            g = dy * w
            dx = rs * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
            if case["residual"]:
                dx = dx + s["dh"].float()
            out["dx"] = dx.to(x.dtype)
            if case["residual"]:
                out["dr"] = out["dx"]
            out["dw"] = (dy * xh).sum(0).to(s["w"].dtype)
            out["db"] = dy.sum(0).to(s["b"].dtype)
        return out


def _best(x, k):
    """Indices of the k largest of each row, ties to the lowest index: by a whole number that orders (value, -index)."""
    bits = (x + 0.0).view(torch.int32)
    order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).to(torch.int64)
    last = x.shape[1] - 1
    key = order * (1 << 32) + (last - torch.arange(x.shape[1], device=x.device))
    return last - (key.topk(k, dim=1).values & 0xFFFFFFFF)


def _plain_lp(s):
    case = s["case"]
    with torch.no_grad():
        x, t = s["logits"].float(), s["targets"]
        d = x - x.amax(-1, keepdim=True)
        e = torch.exp(d)
        total = e.sum(-1, keepdim=True)
        logp = d - torch.log(total)
        p = e / total
        given = t != IGNORE
        at = torch.where(given, t, 0)[:, None]
        zero = torch.zeros((), device=x.device)
        out = dict(log_prob=torch.where(given, logp.gather(1, at)[:, 0], zero))
        if case["entropy"]:
            out["entropy"] = -torch.where(p > 0, p * logp, zero).sum(-1)
        if case["top_k"]:
            out["top_indices"] = _best(x, case["top_k"])
            out["top_log_probs"] = logp.gather(1, out["top_indices"])
        if case["train"]:
            g = torch.where(given, s["g"], zero)[:, None]
            gt = s["gt"] if case["top_k"] else None
            coef = g if gt is None else g + gt.sum(-1, keepdim=True)
            if case["entropy"]:
                coef = coef + s["ge"][:, None] * (logp + out["entropy"][:, None])
            grad = -torch.where(p > 0, p * coef, zero)
            grad.scatter_add_(1, at, g)
            if gt is not None:
                grad.scatter_add_(1, out["top_indices"], gt)
            out["grad"] = grad.to(s["logits"].dtype)
        return out


def _values(codes, scales, signed):
    """What 8-bit codes stand for: the fp32 number whose bits are the magnitude's at bit 19, times 2^127, times the block's scale."""
    c = codes.to(torch.int32)
    mag = ((c & 127 if signed else c) << 19).view(torch.float32) * 2.0 ** 127
    mag = torch.where(c >= 128, -mag, mag) if signed else mag
    return (mag.view(-1, BLOCK) * scales[:, None]).view(-1)


def _encode(values, signed):
    """Codes and scales: magnitudes scaled so that the block's largest has the top code, rounded to nearest even."""
    a = values.abs().view(-1, BLOCK)
    top = TOP_M if signed else TOP_V
    largest = a.amax(1, keepdim=True)
    largest = torch.where(largest < TINY, 0.0, largest)
    inv = torch.where(largest > 0, top / largest, 0.0)
    bits = (a * inv * 2.0 ** -127).view(torch.int32)
    code = (bits + 0x3FFFF + ((bits >> 19) & 1)) >> 19
    code = code.clamp(max=127 if signed else 255)
    if signed:
        code = code + 128 * (values.view(-1, BLOCK) < 0)
    else:
        code = torch.where((a > 0) & (largest > 0), code.clamp(min=1), code)
    return code.to(torch.uint8).view(-1), largest[:, 0] / top


def _plain_adamw(s):
    case, (b1, b2), lr = s["case"], ADAMW["betas"], ADAMW["lr"]
    with torch.no_grad():
        p, g = s["flat_p"].float(), s["flat_g"].float()
        eight = case["bits"] == 8
        m = _values(s["flat_m"], s["scale_m"], True) if eight else s["flat_m"]
        v = _values(s["flat_v"], s["scale_v"], False) if eight else s["flat_v"]
        m = m * b1 + g * (1 - b1)
        v = v * b2 + g * g * (1 - b2)
        s["steps"][:, 0] += 1
        t = s["steps"][0, 0].double()
        p = p * (1 - lr * ADAMW["weight_decay"]) - lr / (1 - b1 ** t) * m / (torch.sqrt(v / (1 - b2 ** t)) + ADAMW["eps"])
        s["flat_p"].copy_(p)
        if not eight:
            s["flat_m"].copy_(m)
            s["flat_v"].copy_(v)
            return dict(p=s["flat_p"], m=s["flat_m"], v=s["flat_v"])
        for k, x in (("m", m), ("v", v)):
            codes, scales = _encode(x, k == "m")
            s["flat_" + k].copy_(codes)
            s["scale_" + k].copy_(scales)
        return dict(p=s["flat_p"], m=_values(s["flat_m"], s["scale_m"], True), v=_values(s["flat_v"], s["scale_v"], False))


# ------------------------------------------------------------------------------------------ the framework's calls

def _own_ln(s):
    from addernetcuda_b200.layernorm import layer_norm
    case = s["case"]
    x, w, b = s["x"], s["w"], s["b"]
    if not case["residual"]:
        y = layer_norm(x, (case["width"],), w, b, EPS)
        if not case["train"]:
            return dict(y=y)
        dx, dw, db = torch.autograd.grad(y, s["leaves"], s["dy"])
        return dict(y=y, dx=dx, dw=dw, db=db)
    y, h = layer_norm(x, (case["width"],), w, b, EPS, residual=s["r"])
    if not case["train"]:
        return dict(y=y, h=h)
    dx, dr, dw, db = torch.autograd.grad((y, h), s["leaves"], (s["dy"], s["dh"]))
    return dict(y=y, h=h, dx=dx, dr=dr, dw=dw, db=db)


def _own_lp(s):
    from addernetcuda_b200.logprobs import token_log_probs
    case = s["case"]
    r = token_log_probs(s["logits"], s["targets"], top_k=case["top_k"], entropy=case["entropy"], ignore_index=IGNORE)
    out = dict(log_prob=r.log_prob)
    if case["entropy"]:
        out["entropy"] = r.entropy
    if case["top_k"]:
        out["top_indices"], out["top_log_probs"] = r.top_indices, r.top_log_probs
    if case["train"]:
        outputs, grads = [r.log_prob], [s["g"]]
        if case["entropy"]:
            outputs.append(r.entropy)
            grads.append(s["ge"])
        if case["top_k"]:
            outputs.append(r.top_log_probs)
            grads.append(s["gt"])
        out["grad"], = torch.autograd.grad(outputs, s["logits"], grads)
    return out


def _own_adamw(s):
    from addernetcuda_b200.optim import adamw_step, adamw_state_values
    if s["case"]["bits"] == 32:
        adamw_step(s["p"], s["g"], s["m"], s["v"], s["steps"], **ADAMW)
        return dict(p=s["flat_p"], m=s["flat_m"], v=s["flat_v"])
    adamw_step(s["p"], s["g"], s["m"], s["v"], s["steps"], exp_avg_scales=s["sm"], exp_avg_sq_scales=s["sv"], **ADAMW)
    return dict(p=s["flat_p"], m=adamw_state_values(s["flat_m"], s["scale_m"], signed=True),
                v=adamw_state_values(s["flat_v"], s["scale_v"], signed=False))


def run(state):
    op = state["case"]["op"]
    if own:
        return _own_ln(state) if op == "ln" else _own_lp(state) if op == "lp" else _own_adamw(state)
    return _plain_ln(state) if op == "ln" else _plain_lp(state) if op == "lp" else _plain_adamw(state)


def work(case):
    size = torch.finfo(TYPES[case["dtype"]]).bits // 8
    if case["op"] == "ln":
        n, d = case["rows"] * case["width"], case["width"]
        wide = torch.finfo(TYPES[case["wtype"]]).bits // 8
        tensors = 2 + 2 * case["residual"] + case["train"] * (2 + case["residual"])      # x, y; r, h; dy, dx; dh
        return dict(bytes=tensors * n * size + (4 if case["train"] else 2) * d * wide, flops=(23 if case["train"] else 8) * n)
    if case["op"] == "lp":
        rows, n, k = case["rows"], case["rows"] * case["classes"], case["top_k"]
        per_row = 8 + 4 + 4 * case["entropy"] + 12 * k + case["train"] * (4 + 4 * case["entropy"] + 4 * k)
        return dict(bytes=n * size * (2 if case["train"] else 1) + rows * per_row, flops=(11 if case["train"] else 5) * n)
    n = sum(_sizes(case))
    # p read and written, g read, both states read and written; states in 8 bits also come back as the values they stand for
    states = 16 if case["bits"] == 32 else 4 + 16 / BLOCK + 8
    return dict(bytes=n * (3 * size + states), flops=16 * n)


# ------------------------------------------------------------------------------------------ 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "ln":
            x, w = s["x"].double(), s["w"].double()
            out = {}
            if case["residual"]:       # the stream is held in its own type, and the norm is taken of what is held
                out["h"] = (x + s["r"].double()).to(s["x"].dtype).double()
                x = out["h"]
            var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
            z = (x - mean) / (var + EPS).sqrt()
            out["y"] = z * w + s["b"].double()
            if case["train"]:
                dy = s["dy"].double()
                dz = dy * w
                n = case["width"]
                dx = (n * dz - dz.sum(-1, keepdim=True) - z * (dz * z).sum(-1, keepdim=True)) / (n * (var + EPS).sqrt())
                out["dx"] = dx + s["dh"].double() if case["residual"] else dx
                if case["residual"]:
                    out["dr"] = out["dx"]
                out["dw"], out["db"] = torch.einsum("ij,ij->j", dy, z), dy.sum(0)
            return out
        if case["op"] == "lp":
            x, t = s["logits"].double(), s["targets"]
            rows = torch.arange(case["rows"], device=DEV)
            given = t != IGNORE
            logp = x - torch.logsumexp(x, -1, keepdim=True)
            p = logp.exp()
            out = dict(log_prob=torch.where(given, logp[rows, t.clamp(min=0)], 0.0))
            entropy = -torch.nan_to_num(p * logp, nan=0.0).sum(-1)
            if case["entropy"]:
                out["entropy"] = entropy
            if case["top_k"]:
                out["top_log_probs"], out["top_indices"] = logp.topk(case["top_k"], -1).values, None
            if case["train"]:
                up = torch.zeros_like(x)       # gradient with respect to the log probabilities, then through the log-softmax
                up[rows[given], t[given]] = s["g"][given].double()
                if case["top_k"]:
                    up.scatter_add_(1, _best(s["logits"].float(), case["top_k"]), s["gt"].double())
                if case["entropy"]:
                    up -= s["ge"].double()[:, None] * p * (logp + 1)
                out["grad"] = up - p * up.sum(-1, keepdim=True)
            return out
        # a code is decided by arithmetic in 32 bits, so what the 8-bit states hold after the step has no value in 64
        eight = case["bits"] == 8
        m = _values(s["flat_m"], s["scale_m"], True).double() if eight else s["flat_m"].double()
        v = _values(s["flat_v"], s["scale_v"], False).double() if eight else s["flat_v"].double()
        g, p = s["flat_g"].double(), s["flat_p"].double()
        (b1, b2), t = ADAMW["betas"], int(s["steps"][0, 0]) + 1
        m = torch.lerp(g, m, b1)
        v = torch.lerp(g.square(), v, b2)
        mhat, vhat = m / (1 - b1 ** t), v / (1 - b2 ** t)
        p = p - ADAMW["lr"] * (ADAMW["weight_decay"] * p + mhat / (vhat.sqrt() + ADAMW["eps"]))
        return dict(p=p, m=None if eight else m, v=None if eight else v)
