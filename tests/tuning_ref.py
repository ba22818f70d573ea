"""64-bit restatements of the tuning operators for the tests."""
import math

import torch


def table(n_pos, dk, theta):
    """(cos, sin) [n_pos, dk / 2, 2] in 64 bits."""
    a = torch.arange(n_pos, dtype=torch.float64)[:, None] * theta ** (-torch.arange(0, dk, 2, dtype=torch.float64) / dk)[None]
    return torch.stack([a.cos(), a.sin()], -1)


def logprob(x, t):
    lse = torch.logsumexp(x, 1)
    return x[torch.arange(x.shape[0], device=x.device), t] - lse, lse


def logprob_back(x, t, lse, g):
    dx = -g[:, None] * torch.exp(x - lse[:, None])
    dx[torch.arange(x.shape[0], device=x.device), t] += g
    return dx


def policy(x, t, old, refp, adv, w, lo, hi, c):
    """Loss per row and d sum(loss) / dx, without grad_scale. old or refp may be None."""
    logp, lse = logprob(x, t)
    r = torch.exp(logp - old) if old is not None else torch.ones_like(logp)
    a, b = r * adv, r.clamp(lo, hi) * adv
    kl, g = torch.zeros_like(logp), torch.where(a <= b, -a, torch.zeros_like(a))
    if refp is not None:
        u = refp - logp
        kl = torch.expm1(u) - u
        g = g - c * torch.expm1(u)
    live = w != 0
    g = torch.where(live, w * g, torch.zeros_like(g))
    loss = torch.where(live, w * (-torch.minimum(a, b) + c * kl), torch.zeros_like(g))
    return {"loss": loss, "logp": logp, "lse": lse, "kl": kl, "g": g, "r": r, "dx": logprob_back(x, t, lse, g)}


def preference(logp, refp, w, seq, beta, eps):
    loss, margin, dlogp = [], [], torch.zeros_like(logp)
    v = w * (logp - refp)
    for i in range(len(seq) // 2):
        a, b, c = seq[2 * i:2 * i + 3]
        z = beta * float(v[a:b].sum() - v[b:c].sum())
        soft = lambda y: math.log1p(math.exp(-abs(y))) + max(y, 0.0)  # noqa: E731
        loss.append((1 - eps) * soft(-z) + eps * soft(z))
        margin.append(z)
        dz = eps - 1 / (1 + math.exp(z))
        dlogp[a:b] = beta * dz * w[a:b]
        dlogp[b:c] = -beta * dz * w[b:c]
    return {"loss": torch.tensor(loss, dtype=torch.float64), "margin": torch.tensor(margin, dtype=torch.float64), "dlogp": dlogp}


def _turn(x, cs, pos, n_rot, sign):
    """x [T, H, dk] with the first n_rot heads rotated; also sum of the two products' magnitudes."""
    c, s = cs[pos].unbind(-1)
    c, s = c[:, None], sign * s[:, None]
    a, b = x[..., 0::2], x[..., 1::2]
    y = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
    size = torch.stack([(a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()], -1).flatten(-2)
    rot = (torch.arange(x.shape[1], device=x.device) < n_rot)[None, :, None]
    return torch.where(rot, y, x), torch.where(rot, size, x.abs())


def qk_forward(x, w, H, cs, pos, n_rot, eps, sizes=False):
    T, dk = x.shape[0], w.numel()
    x = x.reshape(T, H, dk)
    y = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w
    y, size = _turn(y, cs, pos, n_rot, 1.0)
    return (y.flatten(1), size.flatten(1)) if sizes else y.flatten(1)


def qk_backward(dy, x, w, H, cs, pos, n_rot, eps):
    """dx, dw and, for tolerances, (sum of magnitudes behind dx, behind dw)."""
    T, dk = x.shape[0], w.numel()
    x, g = x.reshape(T, H, dk), dy.reshape(T, H, dk)
    g, size = _turn(g, cs, pos, n_rot, -1.0)
    inv = 1 / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    k2 = (g * w * x).mean(-1, keepdim=True) * inv * inv
    big = (size * w.abs() * x.abs()).mean(-1, keepdim=True) * inv * inv
    dx = inv * (g * w - x * k2)
    return dx.flatten(1), (g * x * inv).sum((0, 1)), ((inv * (size * w.abs() + x.abs() * big)).flatten(1),
                                                      (size * x.abs() * inv).sum((0, 1)))


def _mix32(v):
    v = v & 0xFFFFFFFF
    v = ((v ^ (v >> 16)) * 0x9E3779B1) & 0xFFFFFFFF
    v = ((v ^ (v >> 15)) * 0xBB67AE85) & 0xFFFFFFFF
    return v ^ (v >> 16)


def random_bits(i, seed):
    """The 20 bits of element i (int64 tensor) under a step's seed."""
    key = _mix32((seed & 0xFFFFFFFF) + 0x632BE5AB * (seed >> 32))
    return _mix32((i + 0x3C6EF372 * (i >> 32)) ^ key) & 0xFFFFF
