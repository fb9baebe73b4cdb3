"""GPU: the training operators where offsets pass 32 bits: rows on both sides of every 2^31st value against the same rows
alone (bit for bit, where no sum over rows is taken), and the sums over rows against sums of parts in 64 bits.

Tolerance of a sum of T random terms in fp32: f sqrt(T) of the root of their sum of squares (f = 2^-24; partial sums grow
like the root of their number), and one rounding of the type."""
import pytest
import torch

from _util import dev

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def opmx():
    import torch_function as OPMX
    return OPMX


def test_linear_with_more_than_2_31_outputs():
    OPMX = opmx()
    T, K, N = 70001, 72, 32776
    g = torch.Generator(device=dev()).manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, device=dev()).to(BF)
    X, W, B = r(T, K).requires_grad_(True), (r(N, K) / 8).requires_grad_(True), r(N).requires_grad_(True)
    Y = OPMX.linear_epilogue(X, W, B, None, K, N, "silu")
    dY = r(T, N)
    dX, dW, dB = torch.autograd.grad(Y, (X, W, B), dY)
    Wd, Bd = W.detach().double(), B.detach().double()
    at = torch.cat([torch.arange(0, 40), torch.arange(65500, 65560), torch.arange(T - 40, T)]).to(dev())
    H = X.detach()[at].double() @ Wd.t() + Bd
    s = torch.sigmoid(H)
    u = 2.0 ** -8
    assert bool(((Y.detach()[at].double() - H * s).abs() <= u * 1.01 * (H * s).abs() + 1e-4).all())
    dH = dY[at].double() * (s * (1 + H * (1 - s)))
    want = dH @ Wd
    # dH is rounded to bfloat16: four times the root of the sum of squares of those errors
    tol = u * 1.01 * want.abs() + 4 * u * ((dH ** 2) @ (Wd ** 2)).sqrt()
    assert bool(((dX[at].double() - want).abs() <= tol).all())
    sw, qw = torch.zeros(N, K, dtype=torch.float64, device=dev()), torch.zeros(N, K, dtype=torch.float64, device=dev())
    sb, qb = torch.zeros(N, dtype=torch.float64, device=dev()), torch.zeros(N, dtype=torch.float64, device=dev())
    for i in range(0, T, 4096):
        x = X.detach()[i:i + 4096].double()
        H = x @ Wd.t() + Bd
        s = torch.sigmoid(H)
        dH = dY[i:i + 4096].double() * (s * (1 + H * (1 - s)))
        sw += dH.t().contiguous() @ x
        qw += (dH ** 2).t().contiguous() @ (x ** 2)
        sb += dH.sum(0)
        qb += (dH ** 2).sum(0)
    f = 2.0 ** -24 * T ** 0.5
    assert bool(((dW.double() - sw).abs() <= u * 1.01 * sw.abs() + (4 * u + 4 * f) * qw.sqrt()).all())
    # H in 24 bits moves act'(H) by 2^-16 |H| / 2, |H| up to 30 here
    assert bool(((dB.double() - sb).abs() <= u * 1.01 * sb.abs() + (4 * 15 * 2.0 ** -16 + 4 * f) * qb.sqrt()).all())


def test_swiglu_and_pack_with_more_than_2_31_values():
    OPMX = opmx()
    R, D = 150001, 8192
    g = torch.Generator(device=dev()).manual_seed(2)
    x = torch.randn(R, 2 * D, generator=g, device=dev(), dtype=BF).requires_grad_(True)
    y = OPMX.swiglu_checkpoint8(x)
    dy = torch.randn(R, D, generator=g, device=dev(), dtype=BF)
    dx, = torch.autograd.grad(y, x, dy)
    q, code = OPMX.checkpoint8_pack(x)
    u = OPMX.checkpoint8_unpack(q, code, BF)
    for r in (0, 131071, 131072, R - 1):
        one = x.detach()[r:r + 1].clone().requires_grad_(True)
        y1 = OPMX.swiglu_checkpoint8(one)
        assert torch.equal(y1, y[r:r + 1]) and torch.equal(torch.autograd.grad(y1, one, dy[r:r + 1])[0], dx[r:r + 1])
        q1, c1 = OPMX.checkpoint8_pack(one)
        assert torch.equal(q1, q[r:r + 1]) and torch.equal(c1, code[r:r + 1])
        assert torch.equal(OPMX.checkpoint8_unpack(q1, c1, BF), u[r:r + 1])


def test_balance_loss_with_more_than_2_31_scores():
    OPMX = opmx()
    T, E, k = (1 << 23) + 77, 256, 8
    g = torch.Generator(device=dev()).manual_seed(3)
    s = torch.randn(T, E, generator=g, device=dev(), dtype=BF).requires_grad_(True)
    loss, count = OPMX.moe_balance_loss(s, E, k)
    ds, = torch.autograd.grad(loss, s)
    cr, P = torch.zeros(E, dtype=torch.int64, device=dev()), torch.zeros(E, dtype=torch.float64, device=dev())
    for i in range(0, T, 1 << 20):
        z = s.detach()[i:i + (1 << 20)]
        P += torch.softmax(z.double(), -1).sum(0)
        off = OPMX.moe_select_index(z, E, k)[2]
        cr += off[1:] - off[:-1]
    assert torch.equal(cr, count)
    f = cr.double() / (k * T)
    want = E * float((f * P / T).sum())
    # a lane adds T / (256 blocks of 64 tokens) = 512 values in fp32
    assert abs(float(loss.detach()) - want) <= (512 ** 0.5 * 4 + 64) * 2.0 ** -24 * want
    w = E * f / T
    for r in (0, (1 << 23) - 1, 1 << 23, T - 1):
        p = torch.softmax(s.detach()[r].double(), -1)
        dr = p * (w - (p * w).sum())
        tol = 2.0 ** -8 * 1.01 * dr.abs() + 128 * 2.0 ** -24 * p * (w + (p * w).sum())
        assert bool(((ds[r].double() - dr).abs() <= tol).all())


def test_long_sums_of_the_balance_loss_stay_exact():
    """8388608 tokens with k > 8, all with the same scores: 4096 of them in one lane, whose p = 0.0317 is a number that
    rounds the same way at every addition (4096 of them in a row in fp32 are 1015 2^-24 off).  Tolerance: p is off by 64 2^-24;
    64 additions at most are in fp32 in a row (1/2 2^-24 each) and the sums of the lanes and blocks are rounded once each."""
    OPMX = opmx()
    T, E, k = 1 << 23, 65, 9
    row = torch.zeros(E)
    row[1:64:7] = 0.912
    assert int((row > 0).sum()) == k
    s = row.to(dev()).expand(T, E).contiguous()
    loss, count = OPMX.moe_balance_loss(s, E, k)
    assert torch.equal(count.cpu(), T * (row > 0).long())
    want = E * float(torch.softmax(row.double(), 0)[row > 0].sum()) / k
    assert abs(float(loss) - want) <= (64 + 32 + 4) * 2.0 ** -24 * want
