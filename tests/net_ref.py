"""Plain implementations in 64 bits of the acoustic-network operators, and the error their kernels may have.

u = 2^-24 is half a step of float32.  A sum of n products kept in float32 is off by at most n steps of 2 u relative to the sum of the
products' magnitudes, whether an addition rounds or cuts; a result stored in type t by eps(t) / 2 of its value, or half of t's
smallest subnormal step."""
import math

import numpy as np
import torch

U = 2.0 ** -24


def stored(y, dtype):
    """what rounding to `dtype` may cost a value y"""
    tiny = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}[dtype]
    return y.abs() * (torch.finfo(dtype).eps / 2) + tiny


def proj(x, w, bias, adapters, utt_off, slots):
    """(y, bound on a float32 kernel's error before the store) in 64 bits on the CPU; adapters {slot: (a, b, scale)}; rows of no utterance
    are NaN.  An adapter's h may be carried as two bfloat16 parts (cut, then rounded: 2^-17 of h), b as two parts whose smallest
    product is dropped (2^-16)."""
    x, w = x.double().cpu(), w.double().cpu()
    b0 = torch.zeros(w.shape[0], dtype=torch.float64) if bias is None else bias.double().cpu()
    n, k = x.shape
    y = torch.full((n, w.shape[0]), math.nan, dtype=torch.float64)
    err = torch.zeros_like(y)
    if utt_off is None:
        utt_off, slots = [0, n], [-1]
    for u in range(len(utt_off) - 1):
        lo, hi = max(0, utt_off[u]), min(n, utt_off[u + 1])
        if hi <= lo:
            continue
        xs = x[lo:hi]
        y[lo:hi] = xs @ w.t() + b0
        mag = xs.abs() @ w.abs().t() + b0.abs()
        terms, slot = k + 1, slots[u] if slots is not None else -1
        if slot in adapters:
            a, b, s = adapters[slot]
            a, b = a.double().cpu(), b.double().cpu()
            h = s * (xs @ a.t())
            y[lo:hi] += h @ b.t()
            herr = abs(s) * (xs.abs() @ a.abs().t()) * (2 * U * (k + 1)) + h.abs() * (2.0 ** -16 + 2.0 ** -17)
            err[lo:hi] += herr @ b.abs().t()
            mag += h.abs() @ b.abs().t()
            terms += 3 * a.shape[0]
        err[lo:hi] += 2 * U * terms * mag
    return y, err


def act(name, v):
    if name == "relu":
        return torch.where(v < 0, torch.zeros_like(v), v)
    if name == "silu":
        return v * torch.sigmoid(v)
    if name == "gelu":
        return 0.5 * v * torch.erfc(-v / math.sqrt(2.0))
    return v


def gnorm(x, utt_off, groups, weight, bias, eps, name):
    """(y, bound before the store); rows of no utterance are NaN.  The kernel: two subtractions (the mean in two parts), times 1 / sqrt,
    times weight, plus bias: each rounds by u, so 5 u of |z weight| and u of the sum; sums in 64 bits cost (n + 4) 2^-53 of the mean
    square over the variance.  Every activation's slope is below 1.2; its own evaluation is good to 8 u of |v| (erf, exp: 2 steps)."""
    x = x.double().cpu()
    n, c = x.shape
    w = torch.ones(c, dtype=torch.float64) if weight is None else weight.double().cpu()
    b = torch.zeros(c, dtype=torch.float64) if bias is None else bias.double().cpu()
    y = torch.full((n, c), math.nan, dtype=torch.float64)
    err = torch.zeros_like(y)
    for u in range(len(utt_off) - 1):
        lo, hi = max(0, utt_off[u]), min(n, utt_off[u + 1])
        if hi <= lo:
            continue
        g = x[lo:hi].reshape(hi - lo, groups, -1)
        mean = g.mean(dim=(0, 2), keepdim=True)
        var = ((g - mean) ** 2).mean(dim=(0, 2), keepdim=True)
        z = ((g - mean) / torch.sqrt(var + eps)).reshape(hi - lo, c)
        v = z * w + b
        y[lo:hi] = act(name, v)
        count = g.shape[0] * g.shape[2]
        stat = (count + 4) * 2.0 ** -53 * ((g ** 2).mean(dim=(0, 2), keepdim=True) / (var + eps)).expand_as(g).reshape(hi - lo, c)
        shift = (2.0 ** -48 * mean.abs() / torch.sqrt(var + eps)).expand_as(g).reshape(hi - lo, c)
        err[lo:hi] = 1.2 * ((z * w).abs() * (5 * U + stat) + shift * w.abs() + v.abs() * U) + 8 * U * v.abs()
    return y, err


def senones(z, prior, scale, logbase):
    """(scores int16, best, bound on best's error): numpy, 64 bits.  The sum's logarithm: exp is good to 2 steps and its argument to u of
    itself, |z - max z| <= 104 where exp is not 0; float32 sums add n steps at most."""
    z = np.asarray(z.double().cpu() if torch.is_tensor(z) else z, np.float64)
    p = np.zeros(z.shape[1]) if prior is None else np.asarray(prior.double().cpu(), np.float64)
    nan = np.isnan(z).any(axis=1)
    zz = np.where(np.isnan(z), -np.inf, z)
    l = zz - p
    l = np.where(np.isnan(l), -np.inf, l)
    top = l.max(axis=1)
    unit = scale / (math.log(logbase) * 1024)
    with np.errstate(invalid="ignore", over="ignore"):
        d = np.floor((top[:, None] - l) * unit + 0.5)
    d = np.where(l == -np.inf, 32767, np.where(l == top[:, None], 0, d))
    scores = np.minimum(d, 32767).astype(np.int16)
    zmax = zz.max(axis=1)
    safe = np.where(np.isfinite(zmax), zmax, 0.0)
    with np.errstate(invalid="ignore", divide="ignore"):
        lse = safe + np.log(np.exp(zz - safe[:, None]).sum(axis=1))
        best = np.where(zmax == -np.inf, -np.inf, top - lse)
    best = np.where(nan, np.nan, best)
    return scores, best, (z.shape[1] + 110) * 2 * U + np.abs(best) * U
