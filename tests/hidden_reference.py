"""The operators on hidden-state rows in 64 bits (torch), and how far the kernels' outputs may be off.

A rounding is off by half a step at most, relatively: `half(type)`; below a type's normal range by half of its smallest
step, absolutely: `tiny(type)`.  Tolerances count the roundings of each output's own formula.
"""
import numpy as np
import torch

E = 2.0 ** -24  # half a step of binary32


def half(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def out_tolerance(want, dtype, inner):
    """An output of `dtype`, rounded once from a binary32 value that is off by `inner`."""
    return inner + (half(dtype) if dtype != torch.float32 else 0.0) * (want.abs() + inner) + tiny(dtype) + tiny(torch.float32)


def embed(table, token, scale):
    out = torch.zeros((token.numel(), table.shape[1]), dtype=torch.float64, device=table.device)
    live = (token >= 0) & (token < table.shape[0])
    out[live] = table[token[live]].double() * scale
    out[token >= table.shape[0]] = float("nan")
    return out


def embed_tolerance(want, dtype):
    return out_tolerance(want, dtype, E * want.abs())  # one product, rounded to binary32


def embed_grad(grad, token, vocab, scale):
    """The sums, and the sums of the absolute values."""
    live = (token >= 0) & (token < vocab)
    out = torch.zeros((2, vocab, grad.shape[1]), dtype=torch.float64, device=grad.device)
    g = grad[live].double() * scale
    out[0].index_add_(0, token[live], g)
    out[1].index_add_(0, token[live], g.abs())
    return out[0], out[1]


def embed_grad_tolerance(total, want, absolute, scale, dtype):
    """`total` is the sum, `want` what is written (the sum, or that added to what was there)."""
    # at most 32 rows (the kernel takes 16) are added up in 32 bits; the factor and its product; the join's rounding; the addition
    scale32 = abs(float(np.float32(scale)) / scale - 1.0) if scale else 0.0
    inner = (31 + 3) * E * absolute + scale32 * total.abs() + E * want.abs()
    return out_tolerance(want, dtype, inner + tiny(torch.float32))


def rows_of(x, residual=None):
    """h: the sum as the rows' type holds it."""
    if residual is None:
        return x
    return (x.float() + residual.float()).to(x.dtype)


def norm(h, weight, eps):
    f = h.double()
    r = 1.0 / torch.sqrt((f * f).mean(1, keepdim=True) + eps)
    return f * r * (1.0 if weight is None else weight.double())


def norm_tolerance(want, dtype, weight=None):
    # rstd, h rstd and its product with the weight; what underflows in between is multiplied by the weight
    w = 1.0 if weight is None else weight.double().abs()
    return out_tolerance(want, dtype, 3.02 * E * want.abs() + tiny(torch.float32) * (w + 1.0))


def quantized(h, weight):
    """The whole numbers, exactly, and max |h w| (numpy, extended precision: 64 bits hold 254 |h w| and (2k + 1) max)."""
    p = h.double().cpu().numpy().astype(np.longdouble)
    if weight is not None:
        p = p * weight.double().cpu().numpy().astype(np.longdouble)
    a = np.abs(p)
    top = a.max(1, keepdims=True)
    safe = np.where(top > 0, top, 1)
    k = np.floor(127 * a / safe)
    # the quotient may be off by one at a whole number
    k = np.where((k + 1) * top <= 127 * a, k + 1, np.where(k * top > 127 * a, k - 1, k))
    d = 254 * a - (2 * k + 1) * top
    q = np.where((d > 0) | ((d == 0) & (k % 2 == 1)), k + 1, k)
    q = np.where(top > 0, q, 0) * np.sign(p)
    return torch.from_numpy(q.astype(np.int8)), torch.from_numpy(top[:, 0].astype(np.float64))


def norm_grad(h, weight, grad, eps, grad_sum=None):
    f, g = h.double(), grad.double()
    w = torch.ones(f.shape[1], dtype=torch.float64, device=f.device) if weight is None else weight.double()
    m = 1.0 / torch.sqrt((f * f).mean(1, keepdim=True) + eps)
    c = (g * w * f).mean(1, keepdim=True)
    dh = m * (g * w - f * m * m * c)
    if grad_sum is not None:
        dh = dh + grad_sum.double()
    return dh, (g * f * m).sum(0)


def norm_grad_tolerances(h, weight, grad, eps, want, want_weight, dtype):
    f, g = h.double(), grad.double()
    w = 1.0 if weight is None else weight.double()
    m = 1.0 / torch.sqrt((f * f).mean(1, keepdim=True) + eps)
    wg, mean = (g * w).abs(), (g * w * f).abs().mean(1, keepdim=True)
    hk = f.abs() * m * m * mean  # at least |h k|
    # g w, k (its sum's products and its own), h k and the difference; m and its product; the addition
    inner = E * (m * (2 * wg + 4 * hk) + 2 * m * (wg + hk) + want.abs())
    inner = inner + tiny(torch.float32) * (2 + m * (2 + f.abs()))
    terms = (g * f * m).abs().sum(0)
    # m, h m and g h m; a thread adds up a row in 512 at most (the kernel: in 1,024, or up to 768), four waves' sums are added
    n = min(768, -(-h.shape[0] // 512)) + 4
    return out_tolerance(want, dtype, inner), E * ((3 + n) * terms + want_weight.abs()) + tiny(torch.float32) * h.shape[0]


def matmul(q, scale, weight, weight_scale, bias=None):
    """The products, and what the bias is added to (in 64 bits: dot products of 8-bit numbers are whole there)."""
    y = q.double() @ weight.double().t().contiguous()
    y = y * scale.double()[:, None] * weight_scale.double()
    return y if bias is None else y + bias.double(), y


def matmul_tolerance(want, product, dtype):
    # the sum's conversion and two products; the bias' addition
    return out_tolerance(want, dtype, 3.01 * E * product.abs() + E * want.abs() + 2 * tiny(torch.float32))
