"""The AdamW step and its 8-bit states in plain torch operations, each rounded to fp32 by itself: what the kernels are compared with."""
import torch


def decode(codes, scales, signed):
    c = codes.reshape(-1).to(torch.int32)
    mag = ((c & 127 if signed else c) << 19).view(torch.float32) * 2.0 ** 127
    if signed:
        mag = torch.where(c >= 128, -mag, mag)
    return mag * scales.repeat_interleave(256)[:c.numel()]


def encode(values, signed):
    """(codes, scales) of a flat fp32 tensor."""
    n = values.numel()
    x = torch.nn.functional.pad(values, (0, -n % 256)).view(-1, 256)
    top, most = (248.0, 127) if signed else (63488.0, 255)
    largest = x.abs().amax(1, keepdim=True)
    largest = torch.where(largest < 2.0 ** -100, 0.0, largest)
    inv = torch.where(largest > 0, torch.reciprocal(largest) * top, 0.0)
    bits = (x.abs() * inv * 2.0 ** -127).view(torch.int32)
    code = ((bits + 0x3FFFF + ((bits >> 19) & 1)) >> 19).clamp(max=most)
    code = code + 128 * (x < 0) if signed else torch.where((x > 0) & (largest > 0), code.clamp(min=1), code)
    return code.to(torch.uint8).view(-1)[:n], largest[:, 0] * (1.0 / top)


def moments(g, m, v, b1, b2):
    """m and v after a step, in fp32 with every operation rounded."""
    return m * b1 + g * (1 - b1), v * b2 + g * g * (1 - b2)


def update64(p, m, v, t, lr, b1, b2, eps, wd):
    p, m, v = p.double(), m.double(), v.double()
    return p * (1 - lr * wd) - lr / (1 - b1 ** t) * m / ((v / (1 - b2 ** t)).sqrt() + eps)
