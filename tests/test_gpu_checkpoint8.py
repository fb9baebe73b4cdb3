"""GPU: activations in 8 bits (bit for bit against the oracle) and SwiGLU that keeps its input so.

Tolerances: u = eps / 2 of the type for the one rounding of an output.  The logistic function of the 16-bit kernels is
hardware exp2 and reciprocal: its argument is off by |x| 2^-24, so is the result, plus 4 ulp; the fp32 one is within
4 ulp.  Every product adds half an ulp of fp32."""
import pytest
import torch

from _util import dev
from oracle import train_oracle as O

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def opmx():
    import torch_function as OPMX
    return OPMX


def rows(R, D, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, D, generator=g) * torch.exp2(torch.randint(-12, 6, (R, 1), generator=g).float())
    x[:, ::37] *= 30.0
    return x.to(dtype)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def assert_within(got, ref, tol, what):
    got, ref = got.double().cpu(), ref.double()
    bad = ~((got - ref).abs() <= tol)
    assert not bool(bad.any()), "{}: {} of {} off, worst {:.3e}, there allowed {:.3e}".format(
        what, int(bad.sum()), bad.numel(), float((got - ref).abs()[bad].max()), float(tol[bad].min()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 32), (3, 31), (5, 33), (2, 8), (7, 1411), (4, 2816), (300, 64), (2, 3, 96)])
def test_pack_and_unpack_bit_for_bit(dtype, shape):
    OPMX = opmx()
    x = rows(int(torch.tensor(shape[:-1]).prod()), shape[-1], dtype, sum(shape)).view(shape)
    flat = x.reshape(-1, shape[-1]).clone()
    flat[0] = 0.0                                                   # a row of nothing
    if flat.shape[0] > 1:
        flat[1, 0] = torch.finfo(dtype).max                         # the top of the range, where no step is larger
        flat[1, -1] = torch.finfo(dtype).smallest_normal / 2
    if flat.shape[0] > 2:
        flat[2] = flat[2] * 0 + torch.tensor(1.9921875).to(dtype)   # the border where the step doubles
    x = flat.view(shape)
    q, code = OPMX.checkpoint8_pack(x.to(dev()))
    qr, cr = O.pack8(flat)
    assert q.shape == x.shape and code.shape == x.shape[:-1] + ((shape[-1] + 31) // 32,)
    assert torch.equal(q.cpu().view(qr.shape), qr) and torch.equal(code.cpu().view(cr.shape), cr)
    for out in DTYPES:
        y = OPMX.checkpoint8_unpack(q, code, out)
        assert y.dtype == out and torch.equal(y.cpu().view(qr.shape), O.unpack8(qr, cr).to(out))
    held = O.unpack8(qr, cr)
    assert bool(torch.isfinite(OPMX.checkpoint8_unpack(q, code, dtype)).all())
    bound = flat.double().abs().view(flat.shape[0], -1).max(1, keepdim=True).values / 63.5   # one step at the very top
    assert bool(((held - flat.double()).abs() <= bound + 2.0 ** -126).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_and_nans_poison_their_block_alone(dtype):
    OPMX = opmx()
    x = rows(4, 100, dtype, 5)
    x[0, 40], x[1, 99], x[2, 0] = float("inf"), float("nan"), float("-inf")
    q, code = OPMX.checkpoint8_pack(x.to(dev()))
    qr, cr = O.pack8(x)
    assert torch.equal(q.cpu(), qr) and torch.equal(code.cpu(), cr)
    y = OPMX.checkpoint8_unpack(q, code, dtype).cpu()
    assert bool(y[0, 32:64].isnan().all()) and bool(y[1, 96:].isnan().all()) and bool(y[2, :32].isnan().all())
    assert int(y.isnan().sum()) == 32 + 4 + 32


@pytest.mark.parametrize("dtype", DTYPES)
def test_unaligned_and_strided_rows(dtype):
    """Rows at any address: a view one value into its storage (taken as it is, through the C interface), and a
    transposed one through the package."""
    OPMX = opmx()
    from torch_function import _lib
    base = rows(1, 5 * 67 + 1, dtype, 9).flatten().to(dev())
    x = base[1:].view(5, 67)
    q = torch.empty(5 * 67 + 3, dtype=torch.int8, device=dev())[3:].view(5, 67)
    code = torch.empty(5, 3, dtype=torch.uint8, device=dev())
    _lib.check(_lib.lib().opmx_checkpoint8_pack(x.data_ptr(), 5, 67, _lib.dtype_id(x, ""), q.data_ptr(), code.data_ptr(),
                                                _lib.stream_ptr(dev())), "pack")
    qr, cr = O.pack8(x.cpu())
    assert torch.equal(q.cpu(), qr) and torch.equal(code.cpu(), cr)
    t = rows(40, 9, dtype, 3).to(dev()).t()
    q, code = OPMX.checkpoint8_pack(t)
    qr, cr = O.pack8(t.cpu().contiguous())
    assert torch.equal(q.cpu(), qr) and torch.equal(code.cpu(), cr)


def swiglu_tolerances(x, dy, a, g, beta, dtype):
    u, f = half_step(dtype), 2.0 ** -24
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps + 1e-35
    xa, xg = x.double().chunk(2, -1)
    yref = xg * xa * O.logistic(beta * xa)
    ty = yref.abs() * (u + f * (8 + 2 * (beta * xa).abs())) + tiny
    s, d = O.logistic(beta * a), dy.double()
    ba = (beta * a).abs()
    # the two terms of da may cancel, and 1 - s is off by an ulp of 1: measured against their sum of magnitudes
    da = (d * g).abs() * (s * (1 + ba) * (8 + 2 * ba) + ba * s) * f
    dg = (d * a).abs() * s * (8 + 2 * ba) * f
    ref = O.swiglu_backward(a, g, dy, beta)
    return yref, ty, ref, ref.abs() * u * 1.01 + torch.cat([da, dg], -1) * 1.5 + tiny


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,D,beta", [(1, 1, 1.0), (1, 32, 1.0), (3, 33, 1.0), (17, 1411, 1.0), (64, 2816, 1.0),
                                      (2, 7, 1.702), (1000, 40, 0.5), (5, 4096, -1.0)])
def test_swiglu_and_its_gradient(dtype, R, D, beta):
    OPMX = opmx()
    g = torch.Generator().manual_seed(R + D)
    x = (torch.randn(R, 2 * D, generator=g) * 2).to(dtype)
    x[:, ::9] *= 5
    dy = torch.randn(R, D, generator=g).to(dtype)
    xd = x.to(dev()).requires_grad_(True)
    y = OPMX.swiglu_checkpoint8(xd, beta)
    dx, = torch.autograd.grad(y, xd, dy.to(dev()))
    a, gg = O.swiglu_held(x)
    yref, ty, ref, tx = swiglu_tolerances(x, dy, a, gg, beta, dtype)
    assert y.dtype == dtype and dx.dtype == dtype and dx.shape == x.shape
    assert_within(y.detach(), yref, ty, "Y")
    assert_within(dx, ref, tx, "dX")
    # no gradient asked for: the plain operator's very output
    assert torch.equal(OPMX.swiglu_checkpoint8(x.to(dev()), beta), OPMX.swiglu(x.to(dev()), beta))
    with torch.no_grad():
        assert torch.equal(OPMX.swiglu_checkpoint8(xd, beta), y)


def test_swiglu_keeps_the_8_bits_alone():
    """The input may change in place before the backward pass, as only its 8-bit form is used, and what the graph
    holds is 8.25 bits a value."""
    OPMX = opmx()
    x = torch.randn(64, 2 * 640, device=dev(), dtype=torch.bfloat16)
    leaf = x.clone().requires_grad_(True)
    src = leaf * 1.0
    held = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (held.append(t), t)[1], lambda t: t):
        y = OPMX.swiglu_checkpoint8(src)
    assert sum(t.numel() * t.element_size() for t in held) == 64 * 1280 + 64 * 40
    dy = torch.randn_like(y)
    want, = torch.autograd.grad(y, leaf, dy, retain_graph=True)
    src.data.zero_()
    got, = torch.autograd.grad(y, leaf, dy)
    assert torch.equal(got, want)


def test_expanded_gradient_empty_batch_and_leading_dimensions():
    OPMX = opmx()
    x = torch.randn(2, 3, 10, device=dev(), dtype=torch.float32, requires_grad=True)
    y = OPMX.swiglu_checkpoint8(x)
    y.sum().backward()                                              # dY arrives with stride 0
    flat = x.detach().cpu().view(6, 10)
    a, g = O.swiglu_held(flat)
    ones = torch.ones(6, 5)
    _, _, ref, tol = swiglu_tolerances(flat, ones, a, g, 1.0, torch.float32)
    assert y.shape == (2, 3, 5)
    assert_within(x.grad.view(6, 10), ref, tol, "dX")
    e = torch.empty(0, 10, device=dev(), requires_grad=True)
    out = OPMX.swiglu_checkpoint8(e)
    ge, = torch.autograd.grad(out, e, torch.empty(0, 5, device=dev()))
    assert out.shape == (0, 5) and ge.shape == (0, 10)
    q, c = OPMX.checkpoint8_pack(torch.empty(0, 10, device=dev()))
    assert q.shape == (0, 10) and c.shape == (0, 1) and OPMX.checkpoint8_unpack(q, c, torch.float32).shape == (0, 10)


def test_captured_step_replays():
    """Forward and backward in one graph, replayed over new inputs with eager work in between."""
    OPMX = opmx()
    x = torch.randn(37, 2 * 200, device=dev(), dtype=torch.float16, requires_grad=True)
    dy = torch.randn(37, 200, device=dev(), dtype=torch.float16)

    def step():
        y = OPMX.swiglu_checkpoint8(x)
        return y, torch.autograd.grad(y, x, dy)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ys, dxs = step()
    for i in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(37, 400, device=dev()))
        graph.replay()
        torch.cuda.synchronize()
        y, dx = step()
        assert torch.equal(y, ys) and torch.equal(dx, dxs), i


def test_large_rows_past_32_bit_offsets():
    """More than 2^31 values: the last rows still get their own numbers."""
    OPMX = opmx()
    R, D = 150001, 14336
    q = code = None
    x = torch.zeros(R, D, dtype=torch.bfloat16, device=dev())
    x[-3:] = rows(3, D, torch.bfloat16, 1).to(dev())
    q, code = OPMX.checkpoint8_pack(x)
    qr, cr = O.pack8(x[-3:].cpu())
    assert torch.equal(q[-3:].cpu(), qr) and torch.equal(code[-3:].cpu(), cr)
    assert int(q[:-3].count_nonzero()) == 0
    del x
    y = OPMX.checkpoint8_unpack(q, code, torch.bfloat16)
    assert torch.equal(y[-3:].cpu(), O.unpack8(qr, cr).to(torch.bfloat16))


def test_swiglu_gradient_against_differences():
    """Central differences, in float64, of the formula at the held input: h = 2^-10 leaves h^2 / 6 of a third derivative
    below 3 |g| and 2^-43 / h of rounding, the kernel's fp32 arithmetic a few 2^-24 of the terms."""
    OPMX = opmx()
    x, dy = rows(6, 2 * 45, torch.float32, 4), rows(6, 45, torch.float32, 5)
    x = x.clamp(-8, 8)
    xd = x.to(dev()).requires_grad_(True)
    dx, = torch.autograd.grad(OPMX.swiglu_checkpoint8(xd), xd, dy.to(dev()))
    a, g = O.swiglu_held(x)
    held, h = torch.cat([a, g], -1), 2.0 ** -10
    for col in range(held.shape[1]):
        step = torch.zeros_like(held)
        step[:, col] = h
        want = (dy.double() * (O.swiglu(held + step, 1.0) - O.swiglu(held - step, 1.0))).sum(1) / (2 * h)
        i = col % 45
        scale = dy[:, i].double().abs() * (1 + g[:, i].abs()) * (1 + a[:, i].abs())
        assert bool(((dx[:, col].double().cpu() - want).abs() <= scale * (h * h / 2 + 64 * 2.0 ** -24)).all()), col


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("beta", [1.0, 1e6, -1e6])
def test_large_finite_values(dtype, beta):
    """g a, dY g, dY a or beta a beyond fp32 where the output and the gradients are not.  One value per block, whose 8 bits
    are off by 2^-8 and have gradients of their own.  Tolerance: s is off by 8 + |beta a| ulp, three products and
    one rounding; where e^-beta a is below fp32's range, s is 0 instead of 2^-126 at most."""
    OPMX = opmx()
    cases = [(-1e25, 1e25, 1.0), (-3e38, -3e38, 1e30), (-1e20, 3.0, 1e30), (-60.0, 1e38, 1.0), (-20.0, 1e38, 0.5),
             (3e38, 0.25, 0.25), (1e20, 1e18, 1.0), (0.5, 1e38, 1.0), (-200.0, 2e38, 1.0), (0.0, 2e38, 1.0), (1e34, 3.0, 0.5),
             (-1e34, -3.0, 0.5), (1e-5, 1e38, 1.0), (-2e38, 0.0, 0.25)]
    x = torch.tensor([c[:2] for c in cases], dtype=torch.float64).to(dtype)
    dy = torch.tensor([c[2:] for c in cases], dtype=torch.float64).to(dtype)
    xd = x.to(dev()).requires_grad_(True)
    y = OPMX.swiglu_checkpoint8(xd, beta)
    dx, = torch.autograd.grad(y, xd, dy.to(dev()))
    b = torch.tensor(beta, dtype=torch.float32).double()
    u, f, tiny = half_step(dtype), 2.0 ** -24, torch.finfo(dtype).smallest_normal
    xa, xg = x.double().chunk(2, -1)
    ref = O.swiglu(x, b)
    own = lambda a: f * (12 + 2 * (b * a).abs().clamp(max=88.0))
    gone = lambda a: torch.where(b * a < -87, 2.0 ** -126 * a.abs(), 0.0)
    top = float(torch.finfo(dtype).max)
    fits = ref.abs() < top                                       # (with another beta some are beyond the type)
    assert int(fits.sum()) >= 9
    assert_within(y.detach().cpu()[fits], ref[fits], ((own(xa) + u) * 1.01 * ref.abs() + gone(xa) * xg.abs() + tiny)[fits], "Y")
    a, g = O.swiglu_held(x)
    d = dy.double()
    s, ns, ba = O.logistic(b * a), O.logistic(-b * a), (b * a).abs()
    ref = O.swiglu_backward(a, g, dy, b)
    terms = torch.cat([(d * g).abs() * (s + ba * s * ns) * own(a) + f * (d * g).abs() * ba.clamp(max=88.0) * s,
                       (d * a).abs() * s * own(a)], -1)
    # s next to 1: 1 - s has an ulp of 1 of its own, which ba multiplies while 1 - s is not 0 (ba < 17)
    terms += torch.cat([f * (d * g).abs() * torch.where(ba < 17, ba, 0 * ba), 0 * d], -1)
    lost = torch.cat([gone(a) * (1 + ba.clamp(max=104.0)) * (d * g).abs() / a.abs().clamp(min=1e-30), gone(a) * d.abs()], -1)
    fits = ref.abs() < top
    assert int(fits.sum()) >= 20
    assert_within(dx.cpu()[fits], ref[fits], (ref.abs() * u * 1.01 + terms * 1.5 + lost + tiny)[fits], "dX")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,D", [(2048, 2816), (1500, 1411)])
def test_nothing_is_kept_without_gradients(dtype, R, D):
    """Under no_grad, and for an input that asks for no gradient: the plain operator's output bit for bit, as in training,
    and no memory beside it (the 8 bits would be 4 MB and more)."""
    OPMX = opmx()
    x = rows(R, 2 * D, dtype, 6).to(dev())
    leaf = x.clone().requires_grad_(True)
    want = OPMX.swiglu(x, 1.25)
    assert torch.equal(OPMX.swiglu_checkpoint8(leaf, 1.25), want)
    for grads, arg in ((False, leaf), (False, x), (True, x)):
        with torch.set_grad_enabled(grads):
            torch.cuda.synchronize()
            torch.cuda.reset_peak_memory_stats()
            before = torch.cuda.memory_allocated()
            y = OPMX.swiglu_checkpoint8(arg, 1.25)
            assert torch.cuda.max_memory_allocated() - before <= want.numel() * want.element_size() + (1 << 21)  # (whole blocks)
        assert not y.requires_grad and torch.equal(y, want)
        del y
