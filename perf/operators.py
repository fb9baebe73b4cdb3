"""The measured calls of the training and dense-layer operators that stand beside the mixture-of-experts block:

  linear    a matrix product with bias, activation and residual in its epilogue, forward alone (serving) and
            with its gradients (training)
  swiglu    SwiGLU whose input is kept for the backward pass in 8 bits, forward and backward
  balance   the router's balance loss with the tokens per expert, and its gradient

`run` computes each in elementary torch operations in 32 bits, or through the framework's entry points where
`own` is true.

Definitions (t a token, e an expert, all sums over the tokens that the mask keeps)

  linear    H = X W^T + B,  Y = act(H) + R.  act: none, silu H s(H), gelu H Phi(H), gelu_tanh (its tanh form),
            swiglu H[:, D:] * H[:, :D] * s(H[:, :D]) with D = N / 2; s the logistic function.
            dH = dY * act'(H), dX = dH W, dW = dH^T X, dB = sum_t dH, dR = dY.  With checkpoint8, dW is taken with
            the X that its 8-bit form stands for.
  8 bits    blocks of 32 consecutive values of a row (the last one may be shorter).  With m the largest magnitude
            of a block, 2^e the largest power of two not above m, one more if m >= 1.9921875 * 2^e (but not
            beyond the type's largest exponent), the step is 2^max(e - 6, -126) and a value x is held as the
            whole number round-half-even(x / step) in [-127, 127].  Both halves of a SwiGLU row have their own blocks.
  swiglu    Y = g a s(beta a) of the input (a | g); the gradients are taken at the values the 8 bits stand for.
  balance   p = softmax(scores[t]), count[e] = tokens with e among their k largest scores (ties to the lower
            id), f = count / (k n), n the number of tokens kept: loss = E sum_e f_e mean_t p_te, f held constant.
"""
import math
import os
import sys

import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_OPS = None


def _framework():
    global _OPS
    if _OPS is None:
        package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ppl.pmx_amd")
        if package not in sys.path:
            sys.path.insert(0, package)
        import torch_function
        _OPS = torch_function
    return _OPS


# ------------------------------------------------------------------------------------------- cases

def _linear(T, K, N, dtype, act, bias, residual, train, checkpoint8=False):
    return dict(op="linear", T=T, K=K, N=N, dtype=dtype, act=act, bias=bias, residual=residual, train=train,
                checkpoint8=checkpoint8)


def _swiglu(R, D, dtype):
    return dict(op="swiglu", R=R, D=D, dtype=dtype, beta=1.0)


def _balance(T, E, k, dtype, mask):
    return dict(op="balance", T=T, E=E, k=k, dtype=dtype, mask=mask)


def listed():
    return [
        # one token through the gate/up product of a dense feed-forward beside the experts: reading the weights
        dict(name="linear-token", **_linear(1, 4096, 28672, "f16", "swiglu", False, False, False)),
        # a batch of decoded tokens through a down projection that adds the residual stream
        dict(name="linear-decode", **_linear(24, 14336, 4096, "bf16", "none", True, True, False)),
        # the small float32 layer: where a launch counts
        dict(name="linear-small", **_linear(64, 1024, 2816, "f32", "gelu", True, True, False)),
        # a long prompt through the down projection
        dict(name="linear-prompt", **_linear(8192, 14336, 4096, "bf16", "none", False, True, False)),
        # a training step of the gate/up product
        dict(name="linear-train", **_linear(4096, 4096, 28672, "bf16", "swiglu", False, False, True)),
        # a training step on a ragged batch and sizes that fit no tile, its input kept in 8 bits
        dict(name="linear-train-ragged", **_linear(1111, 1001, 1675, "f16", "gelu", True, True, True, True)),
        # the expert rows of a long batch between the two products, in a training step
        dict(name="swiglu-long", **_swiglu(16384, 14336, "bf16")),
        # a ragged batch of odd rows
        dict(name="swiglu-ragged", **_swiglu(1003, 1411, "f16")),
        # the small float32 layer
        dict(name="swiglu-small", **_swiglu(128, 2816, "f32")),
        # one decoding batch: the counts a server watches, latency alone
        dict(name="balance-decode", **_balance(32, 8, 2, "f16", False)),
        # a padded training batch over fine-grained experts
        dict(name="balance-padded", **_balance(8192, 64, 8, "bf16", True)),
        # a long batch over the most experts, logits in 32 bits
        dict(name="balance-long", **_balance(131072, 256, 8, "f32", False)),
    ]


_MOST_FLOPS = 6 * 4096 * 4096 * 28672


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "swiglu", "balance"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "linear":
        K, N = _spread(rng, 64, 14336), _spread(rng, 64, 28672)
        if rng.random() < 0.6:                      # most layers are whole multiples of 64
            K, N = -(-K // 64) * 64, -(-N // 64) * 64
        act = rng.choice(["none", "silu", "gelu", "gelu_tanh", "swiglu"])
        if act == "swiglu":
            N += N % 2
        train = rng.random() < 0.5
        most = min(8192, _MOST_FLOPS // ((6 if train else 2) * K * N))
        return _linear(_spread(rng, 1, max(1, most)), K, N, dtype, act, rng.random() < 0.5, rng.random() < 0.5, train,
                       train and rng.random() < 0.5)
    if op == "swiglu":
        return _swiglu(_spread(rng, 1, 16384), _spread(rng, 32, 14336), dtype)
    E = _spread(rng, 2, 256)
    return _balance(_spread(rng, 1, 131072), E, rng.randint(1, min(8, E)), dtype, rng.random() < 0.5)


def work(case):
    size = _SIZE[case["dtype"]]
    if case["op"] == "linear":
        T, K, N = case["T"], case["K"], case["N"]
        out = N // 2 if case["act"] == "swiglu" else N
        values = T * K + N * K + T * out + (N if case["bias"] else 0) + (T * out if case["residual"] else 0)
        if case["train"]:
            values += T * out + T * K + N * K + (N if case["bias"] else 0)          # dY; dX, dW, dB
        return {"bytes": values * size, "flops": (6 if case["train"] else 2) * T * K * N}
    if case["op"] == "swiglu":
        cells = case["R"] * case["D"]
        return {"bytes": 6 * cells * size, "flops": 20 * cells}                     # X, Y, dY, dX
    cells = case["T"] * case["E"]
    return {"bytes": 2 * cells * size + (case["T"] if case["mask"] else 0), "flops": 10 * cells}


# ------------------------------------------------------------------------------------------ inputs

def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _activations(g, rows, cols, dtype):
    """Activations as layers hand them on: a few features are ten times as large as the others."""
    x = _randn(g, rows, cols)
    x[:, :: max(1, cols // 7)] *= 10.0
    return x.to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(1000003 * (seed + 1))
    dtype = _DT[case["dtype"]]
    s = {"case": case}
    if case["op"] == "linear":
        T, K, N = case["T"], case["K"], case["N"]
        out = N // 2 if case["act"] == "swiglu" else N
        s["X"] = _activations(g, T, K, dtype)
        s["W"] = (_randn(g, N, K) / math.sqrt(K)).to(dtype)
        s["B"] = _randn(g, N).to(dtype) if case["bias"] else None
        s["R"] = _randn(g, T, out).to(dtype) if case["residual"] else None
        if case["train"]:
            s["dY"] = (_randn(g, T, out) * 0.1).to(dtype)
            s["leaves"] = [s[n] for n in ("X", "W", "B", "R") if s[n] is not None]
            for t in s["leaves"]:
                t.requires_grad_(True)
    elif case["op"] == "swiglu":
        s["X"] = _activations(g, case["R"], 2 * case["D"], dtype).requires_grad_(True)
        s["dY"] = (_randn(g, case["R"], case["D"]) * 0.1).to(dtype)
    else:
        T, E = case["T"], case["E"]
        scores = _randn(g, T, E) * 2.0 + _randn(g, E)                               # some experts are liked better
        scores[::3] = torch.round(scores[::3] * 4) / 4                              # and some scores tie
        s["scores"] = scores.to(dtype).requires_grad_(True)
        # a batch of sequences padded on the right, a sixth of it padding
        s["mask"] = (torch.arange(T, device="cuda") % 97 < 81) if case["mask"] else None
        # the loss' weight in the total, times the loss scale that float16 training uses
        s["dloss"] = torch.tensor(0.01 * (65536.0 if case["dtype"] == "f16" else 1.0), device="cuda")
    return s


# ------------------------------------------------------------------------------------- plain forms

def _held_in_8_bits(x):
    """The float32 values that the 8-bit form of the rows of x stands for."""
    rows, cols = x.shape
    emax = 142 if x.dtype == torch.float16 else 254
    pad = -cols % 32
    b = torch.nn.functional.pad(x.float(), (0, pad)).view(rows, -1, 32)
    bits = b.abs().amax(-1, keepdim=True).view(torch.int32)
    e = ((bits + 0x10000) >> 23).clamp(max=emax)
    step = ((e - 6).clamp(min=1) << 23).view(torch.float32)
    return (torch.round(b / step).clamp(-127, 127) * step).view(rows, -1)[:, :cols]


def _act(h, act):
    """-> act(h), and the function that takes the gradient of it to the gradient of h."""
    if act == "none":
        return h, lambda d: d
    if act == "silu":
        s = torch.sigmoid(h)
        return h * s, lambda d: d * (s + h * s * (1 - s))
    if act == "gelu":
        phi = 0.5 * (1 + torch.erf(h * math.sqrt(0.5)))
        return h * phi, lambda d: d * (phi + h * torch.exp(-0.5 * h * h) / math.sqrt(2 * math.pi))
    if act == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        th = torch.tanh(c * (h + 0.044715 * h * h * h))
        return 0.5 * h * (1 + th), lambda d: d * (0.5 * (1 + th) + 0.5 * h * (1 - th * th) * c * (1 + 3 * 0.044715 * h * h))
    a, g = h.chunk(2, -1)
    s = torch.sigmoid(a)
    return g * a * s, lambda d: torch.cat([d * g * (s + a * s * (1 - s)), d * a * s], -1)


def _plain_linear(s):
    c, dtype = s["case"], s["X"].dtype
    X, W = s["X"].detach().float(), s["W"].detach().float()
    H = X @ W.t()
    if s["B"] is not None:
        H = H + s["B"].detach().float()
    Y, back = _act(H, c["act"])
    if s["R"] is not None:
        Y = Y + s["R"].detach().float()
    if not c["train"]:
        return Y.to(dtype)
    dH = back(s["dY"].float())
    Xk = _held_in_8_bits(s["X"].detach()) if c["checkpoint8"] else X
    out = [Y.to(dtype), (dH @ W).to(dtype), (dH.t() @ Xk).to(dtype)]
    if s["B"] is not None:
        out.append(dH.sum(0).to(dtype))
    if s["R"] is not None:
        out.append(s["dY"])
    return out


def _plain_swiglu(s):
    c, X = s["case"], s["X"].detach()
    R, D, beta = c["R"], c["D"], c["beta"]
    a, g = X.float().chunk(2, -1)
    Y = (g * a * torch.sigmoid(beta * a)).to(X.dtype)
    a, g = _held_in_8_bits(X.reshape(2 * R, D)).view(R, 2, D).unbind(1)
    d, sg = s["dY"].float(), torch.sigmoid(beta * a)
    return [Y, torch.cat([d * g * (sg + beta * a * sg * (1 - sg)), d * a * sg], -1).to(X.dtype)]


def _plain_balance(s):
    c, scores = s["case"], s["scores"].detach()
    E, k = c["E"], c["k"]
    z = scores.float()
    keep = torch.ones(c["T"], device=z.device) if s["mask"] is None else s["mask"].float()
    n = keep.sum()
    p = torch.exp(z - z.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True) * keep[:, None]
    ids = torch.sort(z, dim=-1, descending=True, stable=True).indices[:, :k]
    picked = torch.zeros(c["T"], E, device=z.device).scatter_(1, ids, 1.0) * keep[:, None]
    count = picked.sum(0, dtype=torch.float64)
    f = count / (k * n.clamp(min=1))
    loss = E * (f * (p.sum(0, dtype=torch.float64) / n.clamp(min=1))).sum()
    w = (E * f / n.clamp(min=1)).float()
    grad = s["dloss"] * p * (w - (p * w).sum(-1, keepdim=True))
    return [loss.float(), count.long(), grad.to(scores.dtype)]


# ------------------------------------------------------------------------------------ own operators

def _own_linear(s):
    c = s["case"]
    Y = _framework().linear_epilogue(s["X"], s["W"], s["B"], s["R"], c["K"], c["N"], c["act"],
                                     checkpoint8=c["checkpoint8"])
    if not c["train"]:
        return Y
    return [Y.detach(), *torch.autograd.grad(Y, s["leaves"], s["dY"])]


def _own_swiglu(s):
    Y = _framework().swiglu_checkpoint8(s["X"], s["case"]["beta"])
    return [Y.detach(), *torch.autograd.grad(Y, [s["X"]], s["dY"])]


def _own_balance(s):
    c = s["case"]
    loss, count = _framework().moe_balance_loss(s["scores"], c["E"], c["k"], s["mask"])
    return [loss.detach(), count, *torch.autograd.grad(loss, [s["scores"]], s["dloss"])]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"linear": _own_linear, "swiglu": _own_swiglu, "balance": _own_balance}[op](state)
    return {"linear": _plain_linear, "swiglu": _plain_swiglu, "balance": _plain_balance}[op](state)


# ------------------------------------------------------------------------------------------ 64 bits

def _exact_8_bits(x, emax):
    """The values the 8-bit form stands for, from its definition in 64 bits; emax: the type's largest exponent."""
    rows, cols = x.shape
    out = torch.zeros_like(x, dtype=torch.float64)
    for c0 in range(0, cols, 32 * 64):                                              # 64 blocks at a time
        part = x[:, c0:c0 + 32 * 64].double()
        width = part.shape[1]
        full = torch.zeros(rows, -(-width // 32) * 32, dtype=torch.float64, device=x.device)
        full[:, :width] = part
        blocks = full.view(rows, -1, 32)
        m = blocks.abs().max(-1, keepdim=True).values
        frac, e = torch.frexp(m)                                                    # m = frac 2^e, frac in [1/2, 1)
        e = e - 1 + (2 * frac >= 1.9921875).int()
        e = torch.where(m == 0, torch.full_like(e, -126), e)
        e = torch.clamp(torch.clamp(e, max=emax) - 6, min=-126)
        step = ((e.long() + 1023) << 52).view(torch.float64)                        # 2^e, exactly
        out[:, c0:c0 + width] = (torch.clamp(torch.round(blocks / step), -127, 127) * step).view(rows, -1)[:, :width]
    return out


def _logistic(x):
    return 1 / (1 + torch.exp(-x))


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "linear":
            emax = 15 if case["dtype"] == "f16" else 127
            X, W = s["X"].double(), s["W"].double()
            H = torch.mm(X, W.t().contiguous())
            if s["B"] is not None:
                H += s["B"].double()
            act, D = case["act"], case["N"] // 2
            if act == "none":
                Y, slope = H.clone(), torch.ones_like(H)
            elif act == "silu":
                Y, slope = H * _logistic(H), _logistic(H) * (1 + H * _logistic(-H))
            elif act == "gelu":
                cdf = 0.5 * torch.special.erfc(-H / math.sqrt(2.0))
                Y, slope = H * cdf, cdf + H * torch.exp(-H * H / 2) / math.sqrt(2 * math.pi)
            elif act == "gelu_tanh":
                u = 2 * math.sqrt(2 / math.pi) * (H + 0.044715 * H ** 3)            # (1 + tanh(u/2)) / 2 = s(u)
                Y = H * _logistic(u)
                slope = _logistic(u) + H * _logistic(u) * _logistic(-u) * 2 * math.sqrt(2 / math.pi) * (1 + 0.134145 * H ** 2)
            else:
                a, g = H[:, :D], H[:, D:]
                Y = g * a * _logistic(a)
                slope = torch.cat([g * _logistic(a) * (1 + a * _logistic(-a)), a * _logistic(a)], 1)
            if s["R"] is not None:
                Y += s["R"].double()
            if not case["train"]:
                return Y
            dY = s["dY"].double()
            dH = slope.mul_(torch.cat([dY, dY], 1) if act == "swiglu" else dY)
            Xk = _exact_8_bits(s["X"], emax) if case["checkpoint8"] else X
            out = [Y, torch.mm(dH, W), torch.mm(dH.t().contiguous(), Xk)]
            if s["B"] is not None:
                out.append(dH.sum(0))
            if s["R"] is not None:
                out.append(dY)
            return out
        if case["op"] == "swiglu":
            R, D, beta = case["R"], case["D"], case["beta"]
            X = s["X"].double()
            Y = X[:, D:] * X[:, :D] * _logistic(beta * X[:, :D])
            emax = 15 if case["dtype"] == "f16" else 127
            a, g = _exact_8_bits(s["X"][:, :D], emax), _exact_8_bits(s["X"][:, D:], emax)
            dX = torch.empty_like(X)
            del X
            dY, sa = s["dY"].double(), _logistic(beta * a)
            dX[:, D:] = dY * a * sa
            dX[:, :D] = dY * g * sa * (1 + beta * a * _logistic(-beta * a))
            return [Y, dX]
        E, k = case["E"], case["k"]
        z = s["scores"].double()
        rows = torch.arange(case["T"], device=z.device) if s["mask"] is None else torch.nonzero(s["mask"]).flatten()
        n = rows.numel()
        p = torch.softmax(z[rows], -1)
        # an expert is picked where fewer than k beat it: a larger score, or an equal one with a lower id
        count = torch.zeros(E, dtype=torch.int64, device=z.device)
        zr = z[rows]
        for e in range(E):
            own_score = zr[:, e:e + 1]
            beaten = (zr > own_score).sum(1) + (zr[:, :e] == own_score).sum(1)
            count[e] = (beaten < k).sum()
        f = count.double() / max(1, k * n)
        loss = E * (f * p.sum(0)).sum() / max(1, n)
        grad = torch.zeros_like(z)
        grad[rows] = s["dloss"].double() * E / max(1, n) * p * (f - (p @ f)[:, None])
        return [loss, count, grad]
