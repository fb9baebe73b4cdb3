"""CPU oracle of the operators that train beside the mixture-of-experts block, in 64 bits and written from their
formulas: the linear with epilogue and its gradients, activations in 8 bits, SwiGLU on them, the router's
balance loss.  Test infrastructure only."""
import math

import numpy as np
import torch

BLOCK = 32


def logistic(x):
    return torch.special.expit(x)


# ---------------------------------------------------------------- activations in 8 bits

def pack8(X):
    """-> (q int8 [R, D], code uint8 [R, ceil(D/32)]) of the rows of X [R, D], from the definition, block by block."""
    emax = 15 if X.dtype == torch.float16 else 127
    x = X.double().numpy()
    R, D = x.shape
    nb = -(-D // BLOCK)
    q, code = np.zeros((R, D), np.int8), np.zeros((R, nb), np.uint8)
    for b in range(nb):
        part = x[:, b * BLOCK:(b + 1) * BLOCK]
        m = np.abs(part).max(1, initial=0.0)
        bad = ~np.isfinite(part).all(1)
        m = np.where(bad, 0.0, m)
        frac, e = np.frexp(m)                       # m = frac 2^e, frac in [1/2, 1)
        e = e - 1 + (2 * frac >= 1.9921875)
        e = np.where(m == 0, -126, np.minimum(e, emax))
        e = np.maximum(e - 6, -126)
        code[:, b] = np.where(bad, 255, e + 127)
        steps = np.clip(np.rint(np.ldexp(np.where(np.isfinite(part), part, 0.0), -e[:, None])), -127, 127)
        q[:, b * BLOCK:(b + 1) * BLOCK] = np.where(bad[:, None], 0, steps)
    return torch.from_numpy(q), torch.from_numpy(code)


def unpack8(q, code):
    """The held values, float64."""
    e = code.to(torch.int64).repeat_interleave(BLOCK, 1)[:, :q.shape[1]]
    step = torch.from_numpy(np.ldexp(1.0, (e - 127).numpy()))
    return torch.where(e == 255, torch.full((), math.nan, dtype=torch.float64), q.double() * step)


def held8(X):
    return unpack8(*pack8(X))


def swiglu(X, beta):
    a, g = X.double().chunk(2, -1)
    return g * a * logistic(beta * a)


def swiglu_held(X):
    """a, g of X [R, 2D] as their 8 bits hold them."""
    a, g = X.chunk(2, -1)
    return held8(a.contiguous()), held8(g.contiguous())


def swiglu_backward(a, g, dY, beta):
    s, d = logistic(beta * a), dY.double()
    return torch.cat([d * g * s * (1 + beta * a * logistic(-beta * a)), d * a * s], -1)


# ---------------------------------------------------------------- linear with epilogue

def act(H, name):
    """-> act(H), and the factors that take dY to dH (two of them for swiglu), float64."""
    if name == "none":
        return H, (torch.ones_like(H),)
    if name == "silu":
        return H * logistic(H), (logistic(H) * (1 + H * logistic(-H)),)
    if name == "gelu":
        cdf = 0.5 * torch.special.erfc(-H / math.sqrt(2))
        return H * cdf, (cdf + H * torch.exp(-H * H / 2) / math.sqrt(2 * math.pi),)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        s = logistic(2 * c * (H + 0.044715 * H ** 3))
        return H * s, (s + H * s * logistic(-2 * c * (H + 0.044715 * H ** 3)) * 2 * c * (1 + 0.134145 * H ** 2),)
    a, g = H.chunk(2, -1)
    return g * a * logistic(a), (g * logistic(a) * (1 + a * logistic(-a)), a * logistic(a))


def linear_epilogue(X, W, B, R, name):
    """-> (Y, H) in float64; X [T, K]."""
    H = X.double() @ W.double().t()
    if B is not None:
        H = H + B.double()
    Y = act(H, name)[0]
    return (Y if R is None else Y + R.double()), H


def linear_epilogue_backward(X_held, W, H, dY, name):
    """-> dX, dW, dB in float64, for the X that the gradient of W is taken with."""
    dH = torch.cat([f * dY.double() for f in act(H, name)[1]], -1)
    return dH @ W.double(), dH.t() @ X_held.double(), dH.sum(0)


# ---------------------------------------------------------------- balance loss

def picks(scores, k):
    """[T, E] bool: the k largest scores of a row, NaN first, then ties to the lower id."""
    s = scores.double()
    s = torch.where(torch.isnan(s), torch.full_like(s, math.inf), s) + 0.0
    nan = torch.isnan(scores.double())
    T, E = s.shape
    rank = torch.zeros(T, E, dtype=torch.int64)
    for e in range(E):
        beats = (s > s[:, e:e + 1]) & ~(nan[:, e:e + 1] & ~nan) | (nan & ~nan[:, e:e + 1])
        same = (nan & nan[:, e:e + 1]) | (~nan & ~nan[:, e:e + 1] & (s == s[:, e:e + 1]))
        rank[:, e] = beats.sum(1) + same[:, :e].sum(1)
    return rank < k


def softmax_rows(scores):
    """float64 softmax, 0 for a row of -inf alone."""
    s = scores.double()
    empty = (s == -math.inf).all(1, keepdim=True)
    return torch.where(empty, torch.zeros_like(s), torch.softmax(torch.where(empty, torch.zeros_like(s), s), -1))


def balance_loss(scores, k, mask=None):
    """-> loss (float64), count [E] int64, w [E] float64."""
    T, E = scores.shape
    keep = torch.ones(T, dtype=torch.bool) if mask is None else mask
    n = max(1, int(keep.sum()))
    count = picks(scores, k)[keep].sum(0)
    f = count.double() / (k * n)
    loss = E * (f * softmax_rows(scores)[keep].sum(0) / n).sum()
    return loss, count, E * f / n


def balance_loss_backward(scores, w, dloss, mask=None):
    p = softmax_rows(scores)
    g = float(dloss) * p * (w - (p * w).sum(1, keepdim=True))
    return g if mask is None else torch.where(mask[:, None], g, torch.zeros_like(g))
