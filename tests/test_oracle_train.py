"""CPU: the oracle of the training operators against autograd, differences and small cases worked by hand."""
import math

import pytest
import torch

from oracle import train_oracle as O


def test_8_bits_by_hand():
    x = torch.zeros(1, 40)
    x[0, 0], x[0, 1], x[0, 2], x[0, 3] = 1.0, 0.5, 1.0 / 64, 1.5 / 64       # largest 2^0: steps of 2^-6
    x[0, 32] = 1.9921875                                                    # 127.5 / 64: steps of 2^-5
    x[0, 33] = -0.75
    q, code = O.pack8(x)
    assert q[0, :4].tolist() == [64, 32, 1, 2] and code.tolist() == [[127 - 6, 127 - 5]]     # 1.5 rounds to 2
    assert q[0, 32:34].tolist() == [64, -24]
    y = O.unpack8(q, code)
    assert y[0, 0] == 1.0 and y[0, 32] == 2.0 and y[0, 33] == -0.75
    top = torch.full((1, 1), torch.finfo(torch.float16).max, dtype=torch.float16)
    assert float(O.held8(top)) == 127 * 2.0 ** 9                            # no step beyond the type's range
    z = torch.tensor([[0.0, float("inf"), 1.0]])
    assert O.pack8(z)[1].tolist() == [[255]] and bool(O.held8(z).isnan().all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_8_bits_are_within_half_a_step(dtype):
    g = torch.Generator().manual_seed(0)
    x = (torch.randn(50, 100, generator=g) * torch.exp2(torch.randint(-20, 8, (50, 1), generator=g).float())).to(dtype)
    m = torch.nn.functional.pad(x.double().abs(), (0, 28)).view(50, 4, 32).amax(-1).repeat_interleave(32, 1)[:, :100]
    assert bool(((O.held8(x) - x.double()).abs() <= m / 127.5).all())
    assert torch.equal(O.held8(O.held8(x).to(torch.float32)), O.held8(x))   # held values hold


def test_swiglu_backward_is_the_derivative():
    x = torch.randn(5, 12, dtype=torch.float64, requires_grad=True)
    dy = torch.randn(5, 6, dtype=torch.float64)
    for beta in (1.0, 1.702, -0.5):
        g, = torch.autograd.grad(O.swiglu(x, beta), x, dy)
        a, b = x.detach().chunk(2, -1)
        assert torch.allclose(O.swiglu_backward(a, b, dy, beta), g, rtol=1e-12, atol=1e-14)


@pytest.mark.parametrize("act", ["none", "silu", "gelu", "gelu_tanh", "swiglu"])
def test_linear_backward_is_the_derivative(act):
    f64 = torch.float64
    X, W = torch.randn(5, 7, dtype=f64, requires_grad=True), torch.randn(6, 7, dtype=f64, requires_grad=True)
    B = torch.randn(6, dtype=f64, requires_grad=True)
    dY = torch.randn(5, 3 if act == "swiglu" else 6, dtype=f64)
    Y, H = O.linear_epilogue(X, W, B, None, act)
    want = torch.autograd.grad(Y, (X, W, B), dY)
    got = O.linear_epilogue_backward(X.detach(), W.detach(), H.detach(), dY, act)
    assert all(torch.allclose(a, b, rtol=1e-10, atol=1e-12) for a, b in zip(got, want))
    if act == "gelu":
        assert torch.allclose(Y, torch.nn.functional.gelu(H), rtol=1e-12, atol=1e-14)
    if act == "gelu_tanh":
        assert torch.allclose(Y, torch.nn.functional.gelu(H, approximate="tanh"), rtol=1e-12, atol=1e-14)


def test_balance_loss_by_hand_and_by_differences():
    s = torch.tensor([[1.0, 1.0, 0.0], [0.0, 2.0, 2.0], [-math.inf] * 3])
    assert O.picks(s, 1).tolist() == [[True, False, False], [False, True, False], [True, False, False]]
    assert O.picks(s, 2).tolist() == [[True, True, False], [False, True, True], [True, True, False]]
    nan = torch.tensor([[math.inf, math.nan, math.nan, 0.0]])
    assert O.picks(nan, 1).tolist() == [[False, True, False, False]]
    assert O.picks(nan, 3).tolist() == [[True, True, True, False]]
    z = torch.randn(9, 5, dtype=torch.float64, requires_grad=True)
    mask = torch.tensor([True] * 6 + [False] * 3)
    loss, count, w = O.balance_loss(z.detach(), 2, mask)
    assert int(count.sum()) == 12
    f = count.double() / 12
    direct = 5 * (f * torch.softmax(z, -1)[:6].mean(0)).sum()
    assert abs(float(direct) - float(loss)) < 1e-12
    g, = torch.autograd.grad(direct, z)
    assert torch.allclose(O.balance_loss_backward(z.detach(), w, 1.0, mask), g, atol=1e-14)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_8_bits_at_both_ends_of_the_range(dtype):
    """1/127.5 of the block's largest magnitude also where the step may not grow any more; 2^-127 where it may not shrink."""
    info = torch.finfo(dtype)
    top = torch.tensor([info.max, info.max * 0.998, info.max * 0.996, info.max / 2, info.max / 250, -info.max * 0.99], dtype=torch.float64)
    low = torch.tensor([2.0 ** -119, 2.0 ** -120, 2.0 ** -126, 0.4 * 2.0 ** -126, 2.0 ** -127, 1.4 * 2.0 ** -133], dtype=torch.float64)
    for values in (top, low, low[3:]):
        x = values.to(dtype)[None]
        err, m = (O.held8(x) - x.double()).abs().max(), x.double().abs().max()
        assert float(err) <= max(float(m) / 127.5, 2.0 ** -127)
    x = torch.tensor([[0.4 * 2.0 ** -126]])
    assert float(O.held8(x)) == 0.0                                  # all of it, and still within 2^-127
