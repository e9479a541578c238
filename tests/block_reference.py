"""Layer norm, dropout and the Linear layer's products in 64 bits, with bounds on what 32-bit sums and one rounding of a
result may be off by. Written from the formulas; imports nothing of the package.

Bounds: U[dtype] is a type's unit roundoff (2^-8 bf16, 2^-11 fp16, 2^-24 fp32), the largest relative error of one rounding;
a sum of n fp32 terms is off by at most n 2^-24 times the sum of their absolute values in any order, and by the depth
of its tree where that is known."""
import math

import numpy as np
import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -149}  # half a subnormal step
E = 2.0 ** -24


def close(got, want, tol, what=""):
    """got within tol + one rounding to its type of want, everywhere; the same NaN and infinities."""
    dt = got.dtype
    got, want = got.detach().double().cpu(), want.double().cpu()
    tol = tol.double().cpu() if isinstance(tol, torch.Tensor) else tol
    assert got.shape == want.shape, (what, got.shape, want.shape)
    limit = tol + U[dt] * want.abs() + TINY[dt]
    fine = torch.isfinite(want)
    bad = fine & ~((got - want).abs() <= limit)
    bad |= ~fine & ~((got == want) | (torch.isnan(got) & torch.isnan(want)))
    if bad.any():
        i = int(bad.reshape(-1).nonzero()[0])
        off = ((got - want).abs() / (limit + 0 * got)).reshape(-1)[bad.reshape(-1)].max()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside, first at {i}: {got.reshape(-1)[i]} for {want.reshape(-1)[i]}, "
                             f"worst {float(off):.3g} of the bound")


# ---------------------------------------------------------------------------------------- layer norm
def layer_norm(x, w, b, eps):
    """-> y, mean, rstd and the bound of y before its rounding. The sums are trees over lanes of at most 16 serial terms
    (up to 64 here); past the widths that registers hold, dim / 1024 terms."""
    x = x.double()
    D = x.shape[-1]
    mean = x.mean(-1, keepdim=True)
    var = ((x - mean) ** 2).mean(-1, keepdim=True)
    rstd = (var + eps) ** -0.5
    xh = (x - mean) * rstd
    w = torch.ones(D, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros(D, dtype=torch.float64, device=x.device) if b is None else b.double()
    n = 64 + D / 256
    d_mean = n * E * x.abs().mean(-1, keepdim=True)
    # the variance moves by the mean's error squared only (the differences sum to zero), rstd by half its relative error
    tol = w.abs() * (rstd * (d_mean + E * (x - mean).abs()) + xh.abs() * (n * E + rstd ** 2 * d_mean ** 2)) + 4 * E * (xh * w).abs() + 2 * E * b.abs()
    return xh * w + b, mean.squeeze(-1), rstd.squeeze(-1), tol, d_mean.squeeze(-1), rstd.squeeze(-1) * (n * E + (rstd ** 2 * d_mean ** 2).squeeze(-1))


def layer_norm_grads(dy, x, mean, rstd, w, dres):
    """-> dx, dweight, dbias and their bounds before rounding; mean and rstd as given."""
    dy, x, mean, rstd = dy.double(), x.double(), mean.double().unsqueeze(-1), rstd.double().unsqueeze(-1)
    D, rows = x.shape[-1], x.numel() // max(x.shape[-1], 1)
    xh = (x - mean) * rstd
    g = dy if w is None else dy * w.double()
    dx = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    n = 64 + D / 256
    tol = n * E * rstd * (g.abs() + g.abs().mean(-1, keepdim=True) + xh.abs() * (g * xh).abs().mean(-1, keepdim=True))
    if dres is not None:
        dx, tol = dx + dres.double(), tol + 4 * E * dres.double().abs()
    dims = tuple(range(x.dim() - 1))
    m = 64 + rows / 256
    return (dx, (dy * xh).sum(dims) if dims else dy * xh, dy.sum(dims) if dims else dy, tol,
            m * E * ((dy * xh).abs().sum(dims) if dims else (dy * xh).abs()), m * E * (dy.abs().sum(dims) if dims else dy.abs()))


# ---------------------------------------------------------------------------------------- dropout
def philox(counter, key):
    """Philox4x32-10 of python integers (Salmon et al., SC'11): counter four and key two 32-bit words."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def kept(n, p, seed, counter):
    """Which of n elements stay (numpy, unsigned 64-bit)."""
    m = np.uint64(0xFFFFFFFF)
    idx = np.arange((n + 7) // 8, dtype=np.uint64)
    counter &= (1 << 64) - 1
    seed &= (1 << 64) - 1
    c = [idx & m, idx >> np.uint64(32), np.full_like(idx, counter & 0xFFFFFFFF), np.full_like(idx, counter >> 32)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & m, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & m]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    halves = np.stack(c, 1).astype("<u4").view("<u2").reshape(-1)[:n]
    return halves >= threshold(p)


def threshold(p):
    return int(p * 65536 + 0.5)


def scale(p):
    T = threshold(p)
    return float(np.float32(65536) / np.float32(65536 - T)) if T < 65536 else 0.0


# ---------------------------------------------------------------------------------------- linear
def act(z, name):
    if name == "none":
        return z
    if name == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if name == "gelu":
        return z * 0.5 * torch.special.erfc(-z * 2 ** -0.5)
    u = 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3) if name == "gelu_tanh" else z
    return z * torch.sigmoid(u)


def act_grad(z, name):
    if name == "none":
        return torch.ones_like(z)
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * torch.special.erfc(-z * 2 ** -0.5) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = 2 * math.sqrt(2 / math.pi)
        s = torch.sigmoid(c * (z + 0.044715 * z ** 3))
        return s + z * s * (1 - s) * c * (1 + 3 * 0.044715 * z * z)
    s = torch.sigmoid(z)
    return s + z * s * (1 - s)


# What the kernels' activations may be off by in fp32: the erf form's tail is within 0.75e-7 and multiplied by |z| < 6 where
# it counts, the others go through exp2 and rcp of 1 ulp with an argument below 30 off by 2 ulps.
ACT_ERR = 4e-6


def linear_fwd(x, w, bias, residual, name):
    """-> y, pre, and their bounds before rounding."""
    x, w = x.double(), w.double()
    z, size = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        z, size = z + bias.double(), size + bias.double().abs()
    tol_z = (x.shape[-1] + 8) * E * size
    y = act(z, name)
    tol_y = 1.2 * tol_z + (ACT_ERR * (1 + z.abs()) if name != "none" else 0)  # |act'| <= 1.13
    if residual is not None:
        y = y + residual.double()
        tol_y = tol_y + 2 * E * y.abs()
    return y, z, tol_y, tol_z


def linear_bwd(dy, x, w, pre, name, in_pre, in_name):
    """-> dx, dweight, dbias and their bounds before rounding. With an activation, dz is rounded to the operands' type:
    independent errors of at most u |dz|, whose weighted sum stays within 6 u times the root of the sum of squares (over ten of its
    standard deviations)."""
    u = U[x.dtype]
    N, K = w.shape
    shape, M = x.shape, math.prod(x.shape[:-1])
    dy, x, w = dy.double().reshape(M, N), x.double().reshape(M, K), w.double()
    dz = dy
    if name != "none":
        dz = dy * act_grad(pre.double().reshape(M, N), name)
    near = (lambda a, b: 6 * u * ((a * a) @ (b * b)).sqrt()) if name != "none" else (lambda a, b: 0)
    small = ACT_ERR if name != "none" else 0.0
    dx = dz @ w
    tol_x = ((N + 8) * E) * (dz.abs() @ w.abs()) + near(dz, w) + small * (dy.abs() @ w.abs())
    if in_name != "none":
        d = act_grad(in_pre.double().reshape(M, K), in_name)
        tol_x = 1.2 * tol_x + 2 * ACT_ERR * dx.abs()
        dx = dx * d
    dw = dz.t() @ x
    tol_w = ((M + 8) * E) * (dz.abs().t() @ x.abs()) + near(dz.t(), x) + small * (dy.abs().t() @ x.abs())
    one = torch.ones((M, 1), dtype=torch.float64, device=dz.device)
    db = dz.sum(0)
    tol_b = ((M + 8) * E) * dz.abs().sum(0) + small * dy.abs().sum(0) + (near(dz.t(), one).squeeze(1) if name != "none" else 0)
    return dx.reshape(shape), dw, db, tol_x.reshape(shape), tol_w, tol_b
