"""Plain forms of ops/layer_norm.py and ops/adamw.py on the CPU, and how far rounding may take a result from them."""
import math

import torch

E = 2.0 ** -24  # half a step of float32, relative


def layer_norm64(x, residual, weight, bias, eps, dy=None, ds=None):
    """Values in 64 bits, and for each the bound of a kernel's error, from the inputs as they are (any float type)."""
    s = x
    if residual is not None:
        s = (x.float() + residual.float()).to(x.dtype)
    half = torch.finfo(x.dtype).eps / 2
    v = s.double()
    n = v.shape[-1]
    v = v.reshape(-1, n)
    one, zero = torch.ones(n, dtype=torch.float64), torch.zeros(n, dtype=torch.float64)
    w = one if weight is None else weight.double()
    b = zero if bias is None else bias.double()
    mean = v.mean(1, keepdim=True)
    var = (v - mean).square().mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    xhat = (v - mean) * rstd
    # A lane adds at most n / 32 terms one after another, then the lanes' and the warps' sums meet in less than 16 steps.
    length = n / 32 + 16
    # The mean is off by what its sum's roundings make; that moves every centred value, and the variance by its
    # square alone. The variance's own roundings count half in its root. Six more roundings on the way to xhat.
    off_mean = length * E * v.abs().mean(1, keepdim=True)
    off_rstd = 0.5 * ((length + 4) * E + (off_mean * rstd).square()) + 2 * E
    off_xhat = rstd * off_mean + xhat.abs() * (off_rstd + 6 * E)
    y = xhat * w + b
    values = {"s": s, "y": y}
    bounds = {"y": off_xhat * w.abs() + 4 * E * ((xhat * w).abs() + b.abs()) + half * y.abs()}
    if dy is not None:
        d = dy.double().reshape(-1, n)
        g = d * w
        c1, c2 = g.mean(1, keepdim=True), (g * xhat).mean(1, keepdim=True)
        dx = rstd * (g - c1 - xhat * c2)
        off_c1 = (length + 2) * E * g.abs().mean(1, keepdim=True)
        off_c2 = (length + 3) * E * (g * xhat).abs().mean(1, keepdim=True) + (g.abs() * off_xhat).mean(1, keepdim=True)
        size = g.abs() + c1.abs() + (xhat * c2).abs()
        off = rstd * (off_c1 + xhat.abs() * off_c2 + off_xhat * c2.abs() + size * (off_rstd + 6 * E))
        if ds is not None:
            dx = dx + ds.double().reshape(-1, n)
            off = off + 2 * E * (dx.abs() + ds.double().abs().reshape(-1, n))
        values["dx"], bounds["dx"] = dx, off + half * dx.abs()
        # No kernel adds more than 300 rows one after another at the sizes tested.
        chain = min(v.shape[0], 300) + 16
        values["dweight"], values["dbias"] = (d * xhat).sum(0), d.sum(0)
        whalf = torch.finfo(weight.dtype).eps / 2 if weight is not None else E
        bounds["dweight"] = (chain + 3) * E * (d * xhat).abs().sum(0) + (d.abs() * off_xhat).sum(0) + whalf * values["dweight"].abs()
        bounds["dbias"] = chain * E * d.abs().sum(0) + whalf * values["dbias"].abs()
    return values, {k: o + 1e-38 for k, o in bounds.items()}


def check(name, got, want, bound):
    got = got.detach().double().cpu().reshape(want.shape)
    off = (got - want).abs()
    assert torch.isfinite(got).all(), name
    worst = (off / bound).max().item() if off.numel() else 0.0
    assert worst <= 1, "%s is off by %.3g of its bound" % (name, worst)


def mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x9E3779B1) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x6A09E667) & 0xFFFFFFFF
    return x ^ (x >> 16)


def random_bits(first, numel, seed, step):
    at = torch.arange(first, first + numel)
    key = mix((mix((mix(seed) + step) & 0xFFFFFFFF) + (at >> 32)) & 0xFFFFFFFF)
    return mix(((at & 0xFFFFFFFF) + key) & 0xFFFFFFFF)


def encode(x, bits16, never_zero):
    """(codes, scale bytes) of 1-D float32 x, each 32 of which share a scale."""
    n = x.numel()
    pad = torch.nn.functional.pad
    x, bits16 = pad(x, (0, -n % 32)).view(-1, 32), pad(bits16, (0, -n % 32)).view(-1, 32)
    size = x.abs()
    exponent = (size.view(torch.int32).amax(1, keepdim=True) >> 23).clamp(min=8)
    y = size * ((261 - exponent).clamp(min=1) << 23).view(torch.float32)
    small = y < 2.0 ** -6
    t = torch.where(small, y + 2.0 ** -6, y)
    code = ((t.view(torch.int32) + ((bits16.int() << 4) | 8)) >> 20) - torch.where(small, 968, 960)
    if never_zero:
        code = torch.where(size > 0, code.clamp(min=1), code)
    code = code | ((x.view(torch.int32) >> 24) & 0x80)
    code = torch.where(exponent == 255, 0x7F, code)
    return code.view(-1)[:n].to(torch.uint8), torch.where(exponent == 255, 255, exponent - 7).view(-1).to(torch.uint8)


def decode(codes, scales):
    n = codes.numel()
    scale = (scales.int() << 23).view(torch.float32).repeat_interleave(32)[:n]
    return codes.view(torch.float8_e4m3fn).float() * scale


class Adamw:
    """One tensor (1-D, in the order of memory) with its state."""

    def __init__(self, param, bits, seed=0, first=0):
        self.bits, self.seed, self.first, self.step_count = bits, seed, first, 0
        self.type = param.dtype
        self.p = param.detach().float().cpu().reshape(-1).clone()
        n = self.p.numel()
        if bits == 32:
            self.m, self.v = torch.zeros(n), torch.zeros(n)
        else:
            self.m, self.v = torch.zeros(n, dtype=torch.uint8), torch.zeros(n, dtype=torch.uint8)
            self.em, self.ev = (torch.ones(-(-n // 32), dtype=torch.uint8) for _ in range(2))

    def step(self, grad, lr, betas=(0.9, 0.999), eps=1e-8, decay=1e-2, clip=1.0):
        """Moments come out to the bit. Returns (the parameter in 64 bits, the bound of its error); the next step goes on from the
        values that the caller puts into self.p."""
        self.step_count += 1
        t, (b1, b2) = self.step_count, betas
        g = grad.detach().float().cpu().reshape(-1) * torch.tensor(clip, dtype=torch.float32)
        m, v = (self.m, self.v) if self.bits == 32 else (decode(self.m, self.em), decode(self.v, self.ev))
        m = m * b1 + g * (1 - b1)
        v = v * b2 + (g * (1 - b2)) * g
        if self.bits == 32:
            self.m, self.v = m, v
        else:
            h = random_bits(self.first, g.numel(), self.seed, t)
            (self.m, self.em), (self.v, self.ev) = encode(m, h & 0xFFFF, False), encode(v, h >> 16, True)
        root = v.double().sqrt() / math.sqrt(1 - b2 ** t) + eps
        update = lr / (1 - b1 ** t) * m.double() / root
        p = self.p.double()
        want = p * (1 - lr * decay) - update
        # 1 - lr * decay, two products and a difference; the update: the step size (expm1 of a rounded product: 4),
        # root, two products, sum, quotient and product, each within 2 units of the last place (2 E each).
        bound = 4 * E * (p.abs() + want.abs()) + 24 * E * update.abs()
        bound = bound + torch.finfo(self.type).eps / 2 * want.abs() if self.type == torch.bfloat16 else bound
        return want, bound + 1e-38
