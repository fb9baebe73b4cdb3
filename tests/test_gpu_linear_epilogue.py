"""GPU: the linear with bias, activation and residual in its epilogue, and its gradients, against the 64-bit oracle.

Tolerances, u = eps / 2 of the type, f = 2^-24.
  A sum of n products in fp32: every addition rounds by at most f times the partial sum.  Partial sums of random signs
  grow like the root of their number, so the root mean square of the total is f sqrt(n) / 2.4 times the root of the
  sum of squares q of the products; 4 f (8 + sqrt(n)) q is about ten of those.
  Y: that times the largest slope of the activation, its own arithmetic (8 + 2 |exponent|) f, and one rounding u.
  dH: H is kept in 24 bits (float32: 32), a rounding v = 2^-16 (f) that moves act'(H) by v |H| max |act''| (1/2 silu,
  0.8 gelu), and dH is rounded by u.  These errors are independent from value to value: their part of dX and dW is four
  times the root of their sum of squares with each at its bound (about seven standard deviations)."""
import pytest
import torch

from _util import dev
from oracle import train_oracle as O

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16, torch.float32]
ACTS = ["none", "silu", "gelu", "gelu_tanh", "swiglu"]
CURVE = {"none": 0.0, "silu": 0.5, "gelu": 0.8, "gelu_tanh": 0.85}
F = 2.0 ** -24


def opmx():
    import torch_function as OPMX
    return OPMX


def tensors(T, K, N, dtype, act, bias, residual, seed=0):
    g = torch.Generator().manual_seed(seed + T * 7 + K * 3 + N)
    r = lambda *s: torch.randn(*s, generator=g)
    M = N // 2 if act == "swiglu" else N
    X = r(T, K)
    X[:, ::11] *= 4
    return (X.to(dtype), (r(N, K) / K ** 0.5).to(dtype), r(N).to(dtype) if bias else None,
            r(T, M).to(dtype) if residual else None, r(T, M).to(dtype))


def allow(got, ref, tol, what):
    got, ref = got.detach().double().cpu(), ref.double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    bad = ~((got - ref).abs() <= tol)
    assert not bool(bad.any()), "{}: {} of {} off, worst {:.3e} where {:.3e} is allowed, at {}".format(
        what, int(bad.sum()), bad.numel(), float((got - ref).abs()[bad].max()), float(tol.expand_as(bad)[bad].min()),
        bad.nonzero()[0].tolist())


def sum_error(A, B, n):
    """Of fp32 sums over n of products of A [m, n] and B [n, c]."""
    return 4 * F * (8 + n ** 0.5) * ((A.double() ** 2) @ (B.double() ** 2)).sqrt()


def forward_tolerance(X, W, B, R, H, Y, act, dtype):
    u = torch.finfo(dtype).eps / 2
    eh = sum_error(X, W.t(), X.shape[1]) + (0 if B is None else 4 * F * B.double().abs())
    own = 8 + 4 * H.abs()
    if act == "swiglu":
        a, g = H.chunk(2, -1)
        ea, eg = eh.chunk(2, -1)
        e = 1.1 * ea * g.abs() + eg * (a * O.logistic(a)).abs() + F * own.chunk(2, -1)[0] * (g * a * O.logistic(a)).abs()
    else:
        exponent = 1.6 * (H.abs() + 0.045 * H.abs() ** 3) if act == "gelu_tanh" else H.abs() + H ** 2 / 2
        e = 1.2 * eh + (0 if act == "none" else F * (16 + 4 * exponent) * O.act(H, act)[0].abs())
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    return e + (u + 2 * F) * Y.abs() + (0 if R is None else F * R.double().abs()) + tiny


def backward_tolerances(Xh, W, H, dY, act, dtype, ref):
    u = torch.finfo(dtype).eps / 2
    v = F if dtype == torch.float32 else 2.0 ** -16
    d = dY.double().abs()
    K, N, T = W.shape[1], W.shape[0], Xh.shape[0]
    eh = sum_error(Xh, W.t(), K)                 # H itself is a sum
    if act == "swiglu":
        a, g = H.chunk(2, -1)
        ra, rg = (v * a.abs() + eh.chunk(2, -1)[0]), (v * g.abs() + eh.chunk(2, -1)[1])
        arith = F * (16 + 4 * a.abs())
        e = torch.cat([d * (1.1 * rg + 0.5 * g.abs() * ra + arith * g.abs() * (1 + a.abs())),
                       d * (1.1 * ra + arith * a.abs())], -1)
    else:
        arith = 0 if act == "none" else F * (16 + 4 * H.abs()) * (1 + H.abs())
        e = d * (CURVE[act] * (v * H.abs() + eh) + arith)
    dH = torch.cat([f * dY.double() for f in O.act(H, act)[1]], -1)
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    ew = e + (0 if act == "none" else u * dH.abs() + tiny)      # rounded, too
    rss = lambda A, B: 4 * ((A.double() ** 2) @ (B.double() ** 2)).sqrt()
    dX, dW, dB = ref
    return (u * 1.01 * dX.abs() + rss(ew, W) + sum_error(dH, W, N) + tiny,
            u * 1.01 * dW.abs() + rss(ew.t(), Xh) + sum_error(dH.t(), Xh, T) + tiny,
            u * 1.01 * dB.abs() + 4 * (e ** 2).sum(0).sqrt() + 4 * F * (8 + T ** 0.5) * (dH ** 2).sum(0).sqrt() + tiny)


def check(T, K, N, dtype, act, bias=True, residual=True, train=True, checkpoint8=False, seed=0):
    OPMX = opmx()
    X, W, B, R, dY = tensors(T, K, N, dtype, act, bias, residual, seed)
    leaves = [None if t is None else t.to(dev()).requires_grad_(train) for t in (X, W, B, R)]
    Y = OPMX.linear_epilogue(*leaves, K, N, act, checkpoint8=checkpoint8)
    Yr, H = O.linear_epilogue(X, W, B, R, act)
    assert Y.dtype == dtype
    allow(Y, Yr, forward_tolerance(X, W, B, R, H, Yr, act, dtype), "Y")
    if not train:
        return
    wanted = [t for t in leaves if t is not None]
    grads = dict(zip([i for i in range(4) if leaves[i] is not None], torch.autograd.grad(Y, wanted, dY.to(dev()))))
    Xh = O.held8(X) if checkpoint8 else X
    ref = O.linear_epilogue_backward(Xh, W, H, dY, act)
    tols = backward_tolerances(X, W, H, dY, act, dtype, ref)
    for i, what in ((0, "dX"), (1, "dW"), (2, "dB")):
        if i in grads:
            allow(grads[i], ref[i], tols[i], what)
    if residual:
        assert torch.equal(grads[3].cpu(), dY)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("T,K,N", [(1, 64, 64), (1, 256, 512), (3, 100, 36), (7, 33, 10), (64, 200, 130), (130, 129, 258)])
def test_small_and_ragged(dtype, act, T, K, N):
    check(T, K, N, dtype, act)
    check(T, K, N, dtype, act, bias=False, residual=False, checkpoint8=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("T,K,N", [(1, 4096, 512), (2, 1000, 1024), (16, 2048, 96), (17, 777, 514), (33, 2816, 1024),
                                   (300, 1024, 2816), (513, 1001, 834)])
def test_few_rows_and_long_sums(dtype, act, T, K, N):
    check(T, K, N, dtype, act, train=T not in (1, 16))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act,T,K,N", [("none", 1, 4096, 1100), ("gelu", 16, 4104, 1040), ("swiglu", 3, 4120, 1090),
                                       ("swiglu", 16, 264, 16500), ("silu", 7, 264, 16402), ("none", 1, 8 << 10, 513),
                                       ("none", 20, 4096, 1100), ("swiglu", 32, 4099, 1030)])
def test_weights_streamed_by_few_rows(dtype, act, T, K, N):
    check(T, K, N, dtype, act, train=False)
    check(T, K, N, dtype, act, bias=False, residual=False, train=False)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("act,T,K,N", [("none", 3600, 136, 3400), ("swiglu", 3333, 200, 3600), ("gelu", 3500, 77, 3335)])
def test_large_tiles(dtype, act, T, K, N):
    check(T, K, N, dtype, act, checkpoint8=act == "swiglu")


@pytest.mark.parametrize("act,T,K,N", [("gelu", 257, 1024, 1030), ("swiglu", 130, 1100, 640), ("none", 500, 515, 1027),
                                       ("silu", 1025, 260, 1020), ("gelu", 97, 2816, 100), ("none", 2100, 300, 2050)])
def test_float32_in_between(act, T, K, N):
    """Tiles of 32, 64 and 128 rows, with k in ranges and whole."""
    check(T, K, N, torch.float32, act, checkpoint8=act == "silu")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("act,T,K,N", [("swiglu", 3333, 1000, 3600), ("gelu", 3500, 1041, 3335), ("none", 3500, 3600, 1100),
                                       ("silu", 1550, 3500, 3600)])
def test_the_largest_tiles(dtype, act, T, K, N):
    """256 x 256 tiles, which want 16 k-tiles (24 for the gradient of W): forward twice, gradient of X, gradient of W."""
    check(T, K, N, dtype, act)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_large_tiles_in_both_gradients(dtype):
    check(200, 3500, 3600, dtype, "silu")        # dW [3600, 3500]: k is the 200 rows
    check(3500, 3600, 200, dtype, "none")        # dX [3500, 3600]


@pytest.mark.parametrize("dtype", DTYPES)
def test_only_what_is_asked_for(dtype):
    OPMX = opmx()
    X, W, B, R, dY = [t.to(dev()) for t in tensors(40, 72, 56, dtype, "silu", True, True)]
    full = [t.clone().requires_grad_(True) for t in (X, W, B, R)]
    want = torch.autograd.grad(OPMX.linear_epilogue(*full, 72, 56, "silu"), full, dY)
    for i in range(4):
        some = [t.clone().requires_grad_(i == j) for j, t in enumerate((X, W, B, R))]
        got, = torch.autograd.grad(OPMX.linear_epilogue(*some, 72, 56, "silu"), some[i], dY)
        assert torch.equal(got, want[i]), i
    with torch.no_grad():
        Y = OPMX.linear_epilogue(*full, 72, 56, "silu")
    assert not Y.requires_grad and torch.equal(Y, OPMX.linear_epilogue(X, W, B, R, 72, 56, "silu"))


@pytest.mark.parametrize("dtype", DTYPES)
def test_empty_batches(dtype):
    OPMX = opmx()
    W = torch.randn(24, 16, device=dev()).to(dtype).requires_grad_(True)
    B = torch.randn(24, device=dev()).to(dtype).requires_grad_(True)
    for act, M in (("gelu", 24), ("swiglu", 12)):
        X = torch.empty(0, 16, device=dev(), dtype=dtype, requires_grad=True)
        Y = OPMX.linear_epilogue(X, W, B, None, 16, 24, act)
        dX, dW, dB = torch.autograd.grad(Y, (X, W, B), torch.empty(0, M, device=dev(), dtype=dtype))
        assert Y.shape == (0, M) and dX.shape == (0, 16) and not bool(dW.any()) and not bool(dB.any())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K,N", [(64, 64), (61, 35)])
def test_strides_views_and_leading_dimensions(dtype, K, N):
    """Transposed operands, rows that start at odd addresses, an expanded gradient, batches of more dimensions."""
    OPMX = opmx()
    X, W, B, R, dY = tensors(12, K, N, dtype, "silu", True, True)
    want = None
    for form in range(3):
        if form == 0:
            lx, lw, lb, lr = [t.to(dev()).requires_grad_(True) for t in (X, W, B, R)]
            x, w, b, r = lx, lw, lb, lr
        elif form == 1:
            lx, lw, lb, lr = [t.to(dev()) for t in (X.t().contiguous(), W.t().contiguous(), B, R.t().contiguous())]
            for t in (lx, lw, lb, lr):
                t.requires_grad_(True)
            x, w, b, r = lx.t(), lw.t(), lb, lr.t()
        else:
            off = lambda t: torch.cat([t.new_zeros(1), t.flatten()]).to(dev())[1:].view(t.shape)
            x, w, b, r = [off(t).requires_grad_(True) for t in (X, W, B, R)]
        Y = OPMX.linear_epilogue(x.view(3, 4, K) if form != 1 else x, w, b, r.view(3, 4, N) if form != 1 else r, K, N, "silu")
        g = torch.autograd.grad(Y, (x, w, b, r), torch.ones((), device=dev(), dtype=dtype).expand_as(Y))
        Y = Y.reshape(12, N)
        if want is None:
            want = (Y, g)
        else:
            assert torch.equal(Y, want[0]) and all(torch.equal(p, q) for p, q in zip(g, want[1])), form


def test_infinities_stay_in_their_rows():
    """Rows and columns do not leak into others, nor what lies behind the tensors' ends into a tile."""
    OPMX = opmx()
    for dtype in DTYPES:
        for K in (72, 70):
            X, W, B, R, dY = [t.to(dev()) for t in tensors(70, K, 90, dtype, "none", True, True)]
            clean = OPMX.linear_epilogue(X, W, B, R, K, 90)
            Xb, Wb = X.clone(), W.clone()
            Xb[5, 3] = float("inf")
            Wb[11, 7] = float("nan")
            Y = OPMX.linear_epilogue(Xb, Wb, B, R, K, 90)
            keep = torch.ones_like(Y, dtype=torch.bool)
            keep[5], keep[:, 11] = False, False
            assert torch.equal(Y[keep], clean[keep]) and not bool(torch.isfinite(Y[~keep]).any())


def test_difference_quotients_in_float32():
    OPMX = opmx()
    X, W, B, R, dY = tensors(6, 20, 12, torch.float32, "swiglu", True, True)
    lx, lw, lb = [t.to(dev()).requires_grad_(True) for t in (X, W, B)]
    Y = OPMX.linear_epilogue(lx, lw, lb, R.to(dev()), 20, 12, "swiglu")
    g = torch.autograd.grad(Y, (lx, lw, lb), dY.to(dev()))
    f = lambda x, w, b: float((O.linear_epilogue(x, w, b, R, "swiglu")[0] * dY.double()).sum())
    h = 1e-5
    for which, idx in ((0, (2, 3)), (0, (5, 19)), (1, (0, 0)), (1, (11, 7)), (2, (4,)), (2, (9,))):
        args = [X.double(), W.double(), B.double()]
        plus, minus = [a.clone() for a in args], [a.clone() for a in args]
        plus[which][idx] += h
        minus[which][idx] -= h
        d = (f(*plus) - f(*minus)) / (2 * h)
        assert abs(float(g[which][idx]) - d) <= 1e-4 * (1 + abs(d))


def test_a_change_in_place_is_noticed():
    OPMX = opmx()
    X = torch.randn(8, 16, device=dev())
    W = torch.randn(16, 16, device=dev(), requires_grad=True)
    Y = OPMX.linear_epilogue(X, W, None, None, 16, 16, "silu")
    X.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        Y.sum().backward()
    Y = OPMX.linear_epilogue(X, W, None, None, 16, 16, "silu", checkpoint8=True)
    X.add_(1.0)                                                      # only its 8 bits are used
    Y.sum().backward()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("T,K,N", [(5, 128, 256), (200, 1001, 514)])
def test_captured_step_replays(dtype, T, K, N):
    """Two graphs of a training step, replayed in turn over new inputs with eager work in between: the same bits."""
    OPMX = opmx()
    X, W, B, R, dY = [t.to(dev()).requires_grad_(True) for t in tensors(T, K, N, dtype, "swiglu", True, True)]
    dY = dY.detach()

    def step():
        Y = OPMX.linear_epilogue(X, W, B, R, K, N, "swiglu", checkpoint8=True)
        return [Y.detach(), *torch.autograd.grad(Y, (X, W, B), dY)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for i in range(4):
        with torch.no_grad():
            X.copy_(torch.randn(T, K, device=dev()))
        graph, out = graphs[i % 2]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step())), i


def diagonal(dtype, rows):
    """X and a W of ones on the diagonal: H is exactly X, and as large as the type allows."""
    H = torch.tensor(rows, dtype=torch.float64).to(dtype)
    return H, torch.eye(H.shape[1]).to(dtype)


def large(dtype):
    top = float(torch.finfo(dtype).max)
    return [v for v in (0.0, 1.0, 10.5, 31.0, 33.0, 250.0, 6.0e4, 1.0e10, 3.0e18, 1.7e19, 2.0e19, 1.0e20, 1.0e30, 2.0e38)
            if v <= top] + [top]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_slopes_of_large_finite_values(dtype, act):
    """W = 1: H is X, the slopes are those of the formulas, also where h^2 or h^3 is beyond fp32, and every one is finite.
    Tolerance: the slope's own arithmetic as in backward_tolerances, up to |h| = 12 (further out what it is off by is
    h e^-12 and less), one rounding of dH and one of dX, which is a product with one term; e^-x in Y is off by |x| F
    and 0 from x = 88 on."""
    OPMX = opmx()
    v = large(dtype)
    H, W = diagonal(dtype, [v, [-x for x in v]])
    dY = torch.full_like(H, 0.75)
    X = H.to(dev()).requires_grad_(True)
    Y = OPMX.linear_epilogue(X, W.to(dev()), None, None, len(v), len(v), act)
    dX, = torch.autograd.grad(Y, X, dY.to(dev()))
    Yr, (f,) = O.act(H.double(), act)
    assert bool(torch.isfinite(Y).all()) and bool(torch.isfinite(dX).all())
    u, near = torch.finfo(dtype).eps / 2, H.double().abs().clamp(max=12.0)
    tiny = torch.finfo(dtype).smallest_normal
    allow(Y, Yr, (u + 2 * F + F * (16 + 8 * H.double().abs().clamp(max=33.0) ** 2)) * Yr.abs() + tiny, "Y")
    kept = CURVE[act] * near * (F if dtype == torch.float32 else 2.0 ** -16)
    allow(dX, f * 0.75, 2.02 * u * f.abs() * 0.75 + 0.75 * (F * (16 + 4 * near) * (1 + near) + kept) + tiny, "dX")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_swiglu_of_large_finite_values(dtype):
    """g a and dY g beyond fp32 where g a s(a) and the gradients are not.  W = 1.  Tolerance: s is off by 8 + |a| ulp (a fast
    exponential's argument is), three products, the rounding of H in 24 bits, and the roundings of Y, dH and dX; where e^-a is
    below fp32's range (a <= -88), s is 0 instead of 2^-126 at most."""
    OPMX = opmx()
    cases = [(-1e25, 1e25, 1.0), (-3e38, -3e38, 1e30), (-1e20, 3.0, 1e30), (-60.0, 1e38, 1.0), (-60.0, -3e37, 100.0),
             (-20.0, 1e38, 8.0), (3e38, 0.25, 0.5), (1e20, 1e18, 1.0), (0.5, 2e38, 1.0), (-200.0, 3e38, 1.0), (0.0, 3e38, 1.0)]
    a, g, d = [torch.tensor(c, dtype=torch.float64)[:, None] for c in zip(*cases)]
    H, W = diagonal(dtype, torch.cat([a, g], 1).tolist())
    dY = d.to(dtype)
    X = H.to(dev()).requires_grad_(True)
    Y = OPMX.linear_epilogue(X, W.to(dev()), None, None, 2, 2, "swiglu")
    dX, = torch.autograd.grad(Y, X, dY.to(dev()))
    Yr, (fa, fg) = O.act(H.double(), "swiglu")
    a, g = H.double().chunk(2, 1)
    ref = torch.cat([dY.double() * fa, dY.double() * fg], 1)
    u, v = torch.finfo(dtype).eps / 2, F if dtype == torch.float32 else 2.0 ** -16
    own = F * (12 + 2 * a.abs().clamp(max=88.0)) + v * (1 + a.abs().clamp(max=88.0))
    gone = torch.where(a < -87, 2.0 ** -126 * a.abs().clamp(max=104.0), 0.0)       # past 104, e^-a is below 2^-149
    tiny = torch.finfo(dtype).smallest_normal
    assert bool((Yr.abs() < 3e38).all()) and bool((ref.abs() < 3e38).all())       # of the cases above
    allow(Y, Yr, (own + u) * 1.01 * Yr.abs() + gone * g.abs() + tiny, "Y")
    allow(dX, ref, (own + 2 * u) * 1.01 * ref.abs() + gone * dY.double().abs() * torch.cat([g.abs(), 1 + 0 * g], 1) + tiny, "dX")


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_the_last_finite_sums_are_kept_finite(act):
    """X W^T of 2^128 - 2^104, fp32's largest value, out of three bfloat16 terms: Y is an infinity of bfloat16, but the slope is
    1 (0 on the other side) and so dX = dY (0), exactly: W = 1 for the first feature."""
    OPMX = opmx()
    one = [2.0 ** 128 - 2.0 ** 120, 2.0 ** 120 - 2.0 ** 112, 2.0 ** 112 - 2.0 ** 104]
    X = torch.tensor([one, [-v for v in one]], dtype=torch.float64).to(torch.bfloat16)
    assert torch.equal(X.double().sum(1), torch.tensor([2.0 ** 128 - 2.0 ** 104, 2.0 ** 104 - 2.0 ** 128], dtype=torch.float64))
    x = X.to(dev()).requires_grad_(True)
    Y = OPMX.linear_epilogue(x, torch.ones(1, 3, device=dev(), dtype=torch.bfloat16), None, None, 3, 1, act)
    dX, = torch.autograd.grad(Y, x, torch.full((2, 1), 0.75, device=dev(), dtype=torch.bfloat16))
    assert float(Y.detach()[0]) == float("inf") and float(Y.detach()[1]) == 0.0
    assert torch.equal(dX.cpu(), torch.tensor([[0.75] * 3, [0.0] * 3], dtype=torch.bfloat16))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("T,K,N,act", [(40, 72, 56, "silu"), (130, 1001, 515, "none"), (300, 512, 1026, "swiglu"), (64, 4000, 512, "gelu"),
                                       (5, 33, 7, "none"), (700, 256, 4000, "none")])
def test_every_set_of_gradients_in_its_own_workspace(dtype, T, K, N, act):
    """Through the C interface, each in exactly the bytes it asks for: the gradients' bits do not depend on what else is
    wanted, and nothing behind the workspace is written."""
    OPMX = opmx()
    from torch_function import _lib
    L, d, a, p = _lib.lib(), _lib.dtype_id(torch.empty(0, dtype=dtype), ""), _lib.ACTIVATIONS[act], _lib.ptr
    X, W, _, _, dY = [None if t is None else t.to(dev()) for t in tensors(T, K, N, dtype, act, False, False)]
    Y = torch.empty_like(dY)
    H = torch.empty(L.opmx_linear_epilogue_kept_bytes(T, N, d), dtype=torch.uint8, device=dev())
    ws = _lib.workspace(L.opmx_linear_epilogue_workspace_bytes(T, K, N, d, a), dev())
    _lib.check(L.opmx_linear_epilogue(p(X), p(W), None, None, T, K, N, d, a, p(Y), p(H), p(ws), ws.numel(), _lib.stream_ptr(dev())), "")
    q, code = OPMX.checkpoint8_pack(X)
    first = {}
    for wanted in (7, 15, 1, 2, 3, 4, 5, 6, 10, 11, 14):
        dX, dW, dB = (torch.full((T, K), 9.0, dtype=dtype, device=dev()) if wanted & 1 else None,
                      torch.full((N, K), 9.0, dtype=dtype, device=dev()) if wanted & 2 else None,
                      torch.full((N,), 9.0, dtype=dtype, device=dev()) if wanted & 4 else None)
        need = L.opmx_linear_epilogue_gradients_workspace_bytes(T, K, N, d, a, wanted)
        ws = torch.full((need + 4096,), 0x5A, dtype=torch.uint8, device=dev())
        x8 = wanted & 8
        _lib.check(L.opmx_linear_epilogue_gradients(p(dY), None if x8 else p(X), p(q) if x8 else None, p(code) if x8 else None, p(W),
                                                    p(H), T, K, N, d, a, p(dX), p(dW), p(dB), p(ws) if need > 256 else None,
                                                    need if need > 256 else 0, _lib.stream_ptr(dev())), "gradients")
        assert bool((ws[need:] == 0x5A).all()), wanted
        for name, got in (("dX", dX), ("dW8" if x8 else "dW", dW), ("dB", dB)):
            if got is not None:
                assert bool(torch.isfinite(got).all()) and torch.equal(first.setdefault(name, got), got), (wanted, name)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act,T,K,N", [("none", 16, 14335, 128), ("swiglu", 1, 8191, 130), ("gelu", 32, 4095, 700), ("none", 8, 14336, 128),
                                       ("silu", 48, 1536, 9000), ("swiglu", 64, 512, 20000), ("none", 40, 501, 4096),
                                       ("gelu_tanh", 33, 1023, 2100), ("none", 20, 4096, 1024), ("swiglu", 30, 1001, 9000)])
def test_few_rows_by_either_kernel(dtype, act, T, K, N):
    check(T, K, N, dtype, act, train=False)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("act,T,N", [("none", 33, 49300), ("swiglu", 128, 49408), ("none", 129, 49300)])
def test_few_rows_of_many_outputs(dtype, act, T, N):
    """Up to 128 rows in 128 x 128 or 64 x 128 tiles, above that in the largest."""
    check(T, 1032, N, dtype, act, train=False)


@pytest.mark.parametrize("act,T,K,N", [("swiglu", 181, 333, 19264), ("none", 4500, 100, 1024), ("gelu", 1200, 520, 2400)])
def test_float32_past_one_round_of_tiles(act, T, K, N):
    """More 128 x 128 tiles than CUs: those or 64 x 128, whichever fills its last round better."""
    check(T, K, N, torch.float32, act)


@pytest.mark.parametrize("checkpoint8", [False, True])
def test_a_dh_beyond_float16_is_an_infinity(checkpoint8):
    """dH is rounded to the type for the products: where dY act'(H) is past 65504, the row of dX and the rows of dW that it goes
    into are infinities or NaN, as a loss scale that is too large has to show, and no others.  dB is summed unrounded."""
    OPMX = opmx()
    T, K, N = 70, 64, 48
    X, W, B, _, dY = [None if t is None else t.to(dev()) for t in tensors(T, K, N, torch.float16, "swiglu", True, False)]
    W = W.clone()
    W[:N // 2] *= 0.1
    with torch.no_grad():
        B[24 + 3] = 300.0                                            # g of column 3 in every row
    leaves = [t.clone().requires_grad_(True) for t in (X, W, B)]
    run = lambda d: torch.autograd.grad(OPMX.linear_epilogue(*leaves, None, K, N, "swiglu", checkpoint8=checkpoint8), leaves, d)
    dY = dY.clone()
    dY[:, 3] = 0.25
    clean = run(dY)
    big = dY.clone()
    big[5, 3], big[6, 3] = 3000.0, -3832.0                           # dH = 8e5 and -8e5
    _, H = O.linear_epilogue(X.cpu(), W.cpu(), B.cpu(), None, "swiglu")
    fa, fg = O.act(H, "swiglu")[1]
    dH = torch.cat([fa * big.cpu().double(), fg * big.cpu().double()], 1)
    over = dH.abs() > 65520
    assert sorted(over.nonzero().tolist()) == [[5, 3], [6, 3]]
    dX, dW, dB = run(big)
    rows, cols = torch.ones(T, dtype=torch.bool), torch.ones(N, dtype=torch.bool)
    rows[[5, 6]] = False
    cols[[3, 27]] = False                                            # (27: the other half's gradient is finite, but another)
    assert not bool(torch.isfinite(dX[~rows]).any()) and not bool(torch.isfinite(dW[3]).any())
    assert torch.equal(dX[rows], clean[0][rows]) and torch.equal(dW[cols], clean[1][cols])
    assert bool(torch.isfinite(dW[27]).all()) and bool(torch.isfinite(dB).all())
    # H in 24 bits moves the slope by 2^-17 |H|, |H| < 1 in these two rows: 8e5 2^-17 each, and as much again for the arithmetic
    assert abs(float(dB[3]) - float(dH[:, 3].sum())) <= 2 * 2 * 8.1e5 * 2.0 ** -17 + 4096 * 2.0 ** -11
