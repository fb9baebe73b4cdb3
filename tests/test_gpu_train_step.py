"""GPU: the training operators together, as a block trains with them.

    logits = x Wr^T                        router; its balance loss joins the block's
    y = swiglu8(x Wu^T + bu) Wd^T + x      SwiGLU and the down projection keep their inputs in 8 bits

Every stage is checked against the 64-bit oracle on the values that reached it (its input, and the gradient of its
output), with the tolerances its own tests derive.  The gradient of x is the sum of the three paths' gradients: two
roundings of it more."""
import pytest
import torch

from _util import dev
from oracle import train_oracle as O
from test_gpu_checkpoint8 import assert_within, swiglu_tolerances
from test_gpu_linear_epilogue import allow, backward_tolerances, forward_tolerance

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16, torch.float32]
AUX = 0.25


def opmx():
    import torch_function as OPMX
    return OPMX


class Block:
    def __init__(self, T, D, F, E, k, dtype, seed=0):
        g = torch.Generator().manual_seed(seed + T + D + F + E)
        r = lambda *s: torch.randn(*s, generator=g)
        self.T, self.D, self.F, self.E, self.k, self.dtype = T, D, F, E, k, dtype
        self.x = r(T, D).to(dtype)
        self.weights = [(r(E, D) / D ** 0.5).to(dtype), (r(2 * F, D) / D ** 0.5).to(dtype), r(2 * F).to(dtype),
                        (r(D, F) / F ** 0.5).to(dtype)]
        self.dy = r(T, D).to(dtype)
        self.mask = torch.rand(T, generator=g) < 0.8

    def on_gpu(self):
        self.x, self.dy, self.mask = self.x.to(dev()), self.dy.to(dev()), self.mask.to(dev())
        self.weights = [w.to(dev()).requires_grad_(True) for w in self.weights]
        self.x.requires_grad_(True)
        return self

    def forward(self, paths):
        """paths: x for the router, for the up projection and for the residual."""
        OPMX, (wr, wu, bu, wd) = opmx(), self.weights
        logits = OPMX.linear_epilogue(paths[0], wr, None, None, self.D, self.E)
        loss, count = OPMX.moe_balance_loss(logits, self.E, self.k, self.mask)
        h = OPMX.linear_epilogue(paths[1], wu, bu, None, self.D, 2 * self.F)
        a = OPMX.swiglu_checkpoint8(h)
        y = OPMX.linear_epilogue(a, wd, None, paths[2], self.F, self.D, checkpoint8=True)
        return logits, loss, count, h, a, y

    def step(self):
        """-> y, loss, count and the gradients of x and the weights, as new tensors."""
        logits, loss, count, h, a, y = self.forward([self.x] * 3)
        grads = torch.autograd.grad([y, loss], [self.x, *self.weights], [self.dy, torch.full_like(loss, AUX)])
        return [y.detach(), loss.detach(), count, *grads]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,D,F,E,k", [(1, 64, 96, 8, 2), (37, 100, 66, 5, 1), (300, 257, 190, 64, 8), (600, 512, 1024, 256, 8)])
def test_each_stage_of_a_step(dtype, T, D, F, E, k):
    b = Block(T, D, F, E, k, dtype).on_gpu()
    paths = [b.x.detach().clone().requires_grad_(True) for _ in range(3)]
    logits, loss, count, h, a, y = b.forward(paths)
    for t in (logits, h, a):
        t.retain_grad()
    torch.autograd.backward([y, loss], [b.dy, torch.full_like(loss, AUX)])
    x, dy, mask = b.x.detach().cpu(), b.dy.cpu(), b.mask.cpu()
    wr, wu, bu, wd = [w.detach().cpu() for w in b.weights]
    c = lambda t: t.detach().cpu()

    def linear(X, W, B, R, Y, dY, grads, held=None):
        Yr, H = O.linear_epilogue(X, W, B, R, "none")
        allow(Y, Yr, forward_tolerance(X, W, B, R, H, Yr, "none", dtype), "Y")
        ref = O.linear_epilogue_backward(X if held is None else held, W, H, dY, "none")
        for got, want, tol, what in zip(grads, ref, backward_tolerances(X, W, H, dY, "none", dtype, ref), ("dX", "dW", "dB")):
            if got is not None:
                allow(got, want, tol, what)

    linear(x, wr, None, None, logits, c(logits.grad), (paths[0].grad, b.weights[0].grad, None))
    lr, cr, w = O.balance_loss(c(logits), k, mask)
    assert torch.equal(count.cpu(), cr)
    assert abs(float(c(loss)) - float(lr)) <= 256 * 2.0 ** -24 * float(lr)
    gr = O.balance_loss_backward(c(logits), w, AUX, mask)
    p, info = O.softmax_rows(c(logits)), torch.finfo(dtype)
    allow(logits.grad, gr, gr.abs() * info.eps / 2 + 128 * 2.0 ** -24 * AUX * p * (w + (p * w).sum(1, keepdim=True)) * 1.01
          + info.smallest_normal * info.eps, "gradient of the scores")
    linear(x, wu, bu, None, h, c(h.grad), (paths[1].grad, b.weights[1].grad, b.weights[2].grad))
    yr, ty, ref, tx = swiglu_tolerances(c(h), c(a.grad), *O.swiglu_held(c(h)), 1.0, dtype)
    assert_within(c(a), yr, ty, "swiglu")
    assert_within(c(h.grad), ref, tx, "swiglu's gradient")
    linear(c(a), wd, None, x, y, dy, (a.grad, b.weights[3].grad, None), held=O.held8(c(a)))
    assert torch.equal(paths[2].grad, b.dy)

    whole = b.step()
    assert torch.equal(whole[0], y) and torch.equal(whole[1], loss) and torch.equal(whole[2], count)
    parts = [c(t.grad).double() for t in paths]
    bound = info.eps / 2 * 1.01 * 2 * sum(t.abs() for t in parts)
    allow(whole[3], sum(parts), bound, "sum of the paths")
    for got, t in zip(whole[4:], b.weights):
        assert torch.equal(got, t.grad)


@pytest.mark.parametrize("dtype", DTYPES)
def test_on_another_stream_beside_a_step_on_this_one(dtype):
    """Two steps at once on two streams: neither meets the other's workspaces."""
    one, two = Block(200, 256, 320, 16, 2, dtype, 1).on_gpu(), Block(129, 384, 160, 64, 8, dtype, 2).on_gpu()
    want = [one.step(), two.step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        with torch.cuda.stream(side):
            got_two = two.step()
        got_one = one.step()
        torch.cuda.synchronize()
        for got, ref in zip(got_one + got_two, want[0] + want[1]):
            assert torch.equal(got, ref)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", [1, 150])
def test_two_captured_steps_replayed_in_turn(dtype, T):
    blocks = [Block(T, 192, 256, 32, 4, dtype, s).on_gpu() for s in (1, 2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for b in blocks:
            b.step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for b in blocks:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = b.step()
        graphs.append((graph, out))
    for i in range(6):
        b, (graph, out) = blocks[i % 2], graphs[i % 2]
        with torch.no_grad():
            b.x.copy_(torch.randn_like(b.x))
            b.mask.copy_(torch.rand(T, device=dev()) < 0.6)
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(out, b.step()):
            assert torch.equal(got, want), i


def test_a_few_steps_of_descent():
    """Plain SGD over the block runs, moves every weight and stays finite."""
    b = Block(96, 128, 160, 16, 2, torch.float32).on_gpu()
    before = [w.detach().clone() for w in b.weights]
    for _ in range(3):
        grads = b.step()[4:]
        with torch.no_grad():
            for w, g in zip(b.weights, grads):
                w -= 0.01 * g
    for w, old in zip(b.weights, before):
        assert bool(torch.isfinite(w).all()) and not torch.equal(w, old)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_nothing_is_kept_without_gradients(dtype):
    """Under no_grad, weights that ask for gradients cost no memory beside the output."""
    OPMX = opmx()
    T, K, N = 512, 64, 2048
    x, w = torch.randn(T, K, device=dev(), dtype=dtype), torch.randn(N, K, device=dev(), dtype=dtype, requires_grad=True)
    kept = []
    for grads in (False, True):
        with torch.set_grad_enabled(grads):
            torch.cuda.synchronize()
            before = torch.cuda.memory_allocated()
            y = OPMX.linear_epilogue(x, w, None, None, K, N, "gelu", checkpoint8=True)
            kept.append(torch.cuda.memory_allocated() - before - y.numel() * y.element_size())
        if not grads:
            want = y
        assert y.requires_grad == grads and torch.equal(y, want)
    assert kept[0] <= 512 and kept[1] >= T * N            # X W^T, a byte a value at least
