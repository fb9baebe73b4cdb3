"""GPU: balance loss, tokens per expert and the gradient of the scores against the 64-bit oracle.

Tolerances.  p = exp(z - m) / sum in fp32: z - m and exp are off by |z - m| + 2 ulp (|z - m| <= 40 here), the sum of up
to 256 terms and the division by 20 more: 64 * 2^-24 relative.  Sums over at most a few hundred tokens per lane add 160
ulp: the loss is within 256 * 2^-24.  The gradient is a difference of two terms, each off by less than 128 * 2^-24, and
is rounded once."""
import pytest
import torch

from _util import dev, tie_heavy_scores
from oracle import train_oracle as O

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def opmx():
    import torch_function as OPMX
    return OPMX


def check(scores, k, mask=None, dloss=1.0, strided=False):
    OPMX = opmx()
    T, E = scores.shape
    sd = scores.to(dev())
    if strided:
        sd = torch.stack([sd, sd], -1)[..., 0]
    sd = sd.requires_grad_(True)
    md = None if mask is None else mask.to(dev())
    loss, count = OPMX.moe_balance_loss(sd, E, k, md)
    g, = torch.autograd.grad(loss, sd, torch.tensor(float(dloss), device=dev()))
    lr, cr, w = O.balance_loss(scores, k, mask)
    gr = O.balance_loss_backward(scores, w, dloss, mask)
    assert loss.dtype == torch.float32 and loss.dim() == 0 and count.dtype == torch.int64 and not count.requires_grad
    assert torch.equal(count.cpu(), cr)
    assert abs(float(loss) - float(lr)) <= 256 * 2.0 ** -24 * float(lr)
    p = O.softmax_rows(scores)
    terms = abs(dloss) * p * (w + (p * w).sum(1, keepdim=True))
    info = torch.finfo(scores.dtype)
    tol = gr.abs() * info.eps / 2 + 128 * 2.0 ** -24 * terms * 1.01 + info.smallest_normal * info.eps
    assert g.dtype == scores.dtype and g.shape == scores.shape
    bad = ~((g.double().cpu() - gr).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), float((g.double().cpu() - gr).abs()[bad].max()))
    if mask is not None:
        assert not bool(g.cpu()[~mask].any())
    return loss, count, g


def logits(T, E, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(T, E, generator=g) * 2 + torch.randn(E, generator=g)).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 2), (32, 8, 2), (63, 2, 2), (64, 64, 8), (65, 65, 8), (1000, 7, 3),
                                   (777, 60, 6), (513, 256, 8), (100, 255, 1), (40, 256, 32), (50, 33, 32), (4097, 16, 4),
                                   (300, 128, 9), (9001, 8, 2)])
def test_matches_the_oracle(dtype, T, E, k):
    check(logits(T, E, dtype, T + E + k), k, dloss=3.0)
    g = torch.Generator().manual_seed(T)
    check(logits(T, E, dtype, T + 1), k, mask=torch.rand(T, generator=g) < 0.7, dloss=-0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("E,k", [(8, 2), (16, 4), (64, 8), (65, 7), (200, 8), (256, 32), (6, 5)])
def test_ties_go_to_the_lower_id_as_in_moe_select(dtype, E, k):
    OPMX = opmx()
    s = tie_heavy_scores(701, E, dtype, 3)
    s[5] = 0.0                                       # everything ties
    s[6, ::2] = -0.0
    _, count, _ = check(s, k)
    off = OPMX.moe_select_index(s.to(dev()), E, k)[2]
    assert torch.equal(off[1:] - off[:-1], count)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("E", [8, 40, 256])
def test_masked_experts_and_empty_rows(dtype, E):
    s = logits(300, E, dtype, 11)
    s[:, 3] = float("-inf")                          # an expert that is switched off
    s[7] = float("-inf")                             # a row with nothing left
    s[8] = torch.finfo(dtype).min
    s[9, :-1] = float("-inf")
    _, _, g = check(s, 2, dloss=100.0)
    assert not bool(g[7].any()) and bool(torch.isfinite(g).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_nan_and_infinity(dtype):
    """A token that counts makes the loss NaN and leaves the other rows' gradients alone; behind the mask it is nothing."""
    OPMX = opmx()
    s = logits(100, 16, dtype, 2)
    s[10, 4], s[20, 5] = float("nan"), float("inf")
    sd = s.to(dev()).requires_grad_(True)
    loss, count = OPMX.moe_balance_loss(sd, 16, 4)
    g, = torch.autograd.grad(loss, sd)
    assert bool(loss.isnan()) and torch.equal(count.cpu(), O.picks(s, 4).sum(0))
    rows = g.isnan().any(1).nonzero().flatten().tolist()
    assert rows == [10, 20]
    mask = torch.ones(100, dtype=torch.bool)
    mask[10] = mask[20] = False
    clean = s.clone()
    clean[10] = clean[20] = 0.0
    a = OPMX.moe_balance_loss(sd, 16, 4, mask.to(dev()))
    b = OPMX.moe_balance_loss(clean.to(dev()), 16, 4, mask.to(dev()))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    g, = torch.autograd.grad(a[0], sd)
    assert bool(torch.isfinite(g).all()) and not bool(g[10].any()) and not bool(g[20].any())


def test_no_tokens_and_no_token_kept():
    OPMX = opmx()
    for T in (0, 5):
        s = torch.randn(T, 8, device=dev(), requires_grad=True)
        m = torch.zeros(T, dtype=torch.bool, device=dev())
        loss, count = OPMX.moe_balance_loss(s, 8, 2, m)
        g, = torch.autograd.grad(loss, s)
        assert float(loss) == 0.0 and not bool(count.any()) and g.shape == s.shape and not bool(g.any())


def test_even_router_scores_one_and_leading_dimensions():
    OPMX = opmx()
    eye = torch.eye(8, device=dev()).repeat(6, 1) * 3
    loss, count = OPMX.moe_balance_loss(eye.view(2, 24, 8), 8, 1)
    assert abs(float(loss) - 1.0) < 1e-6 and count.tolist() == [6] * 8


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_scores_and_unaligned_rows(dtype):
    check(logits(70, 24, dtype, 4), 3, strided=True)
    OPMX = opmx()
    base = logits(1, 24 * 9 + 1, dtype, 5).flatten().to(dev())
    s = base[1:].view(9, 24)
    loss, count = OPMX.moe_balance_loss(s, 24, 3)
    ref = OPMX.moe_balance_loss(s.clone(), 24, 3)
    assert torch.equal(count, ref[1]) and abs(float(loss) - float(ref[0])) <= 256 * 2.0 ** -24 * float(ref[0])


def test_gradient_against_differences():
    """float64 differences of the oracle's loss with the counts held, against the kernel's gradient."""
    s = logits(12, 16, torch.float32, 8)
    _, _, g = check(s, 4)
    _, count, _ = O.balance_loss(s, 4)
    f = count.double() / (4 * 12)
    loss = lambda z: 16 * (f * torch.softmax(z, -1).sum(0) / 12).sum()
    h = 1e-5
    for t, e in [(0, 0), (3, 7), (11, 15), (5, 2)]:
        zp, zm = s.double().clone(), s.double().clone()
        zp[t, e] += h
        zm[t, e] -= h
        d = float(loss(zp) - loss(zm)) / (2 * h)
        assert abs(float(g[t, e]) - d) <= 1e-7 + 1e-5 * abs(d)


def test_same_bits_every_time_and_on_another_stream():
    OPMX = opmx()
    s = logits(20000, 64, torch.bfloat16, 6).to(dev()).requires_grad_(True)

    def step():
        loss, count = OPMX.moe_balance_loss(s, 64, 8)
        return loss, count, torch.autograd.grad(loss, s)[0]

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, second))


@pytest.mark.parametrize("T", [16, 5000])
def test_captured_step_replays(T):
    OPMX = opmx()
    s = torch.randn(T, 32, device=dev(), requires_grad=True)
    mask = torch.rand(T, device=dev()) < 0.5

    def step():
        loss, count = OPMX.moe_balance_loss(s, 32, 4, mask)
        return loss, count, torch.autograd.grad(loss, s)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):                               # two graphs, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for i in range(4):
        with torch.no_grad():
            s.copy_(torch.randn(T, 32, device=dev()))
            mask.copy_(torch.rand(T, device=dev()) < 0.5)
        graph, out = graphs[i % 2]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step())), i


@pytest.mark.parametrize("E", [2, 3, 8, 31])
def test_no_gradient_where_every_expert_is_picked(E):
    """k = E: all w are the same float, the gradient is zero, and what rounding leaves of it is of second order: p has a
    relative error of 64 * 2^-24, and so has the mean that is taken away."""
    OPMX = opmx()
    s = logits(500, E, torch.float32, E).to(dev()).requires_grad_(True)
    loss, count = OPMX.moe_balance_loss(s, E, E)
    g, = torch.autograd.grad(loss, s)
    assert bool((count == 500).all())
    assert float(g.abs().max()) <= 2 * (64 * 2.0 ** -24) ** 2 / 500


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,E,k", [(64, 256, 32), (65, 256, 32), (129, 128, 9), (4096, 100, 9), (4500, 251, 17), (33, 64, 12),
                                   (64, 64, 12), (700, 40, 10), (9000, 9, 9), (5000, 16, 16)])
def test_many_picks_from_one_block_to_all(dtype, T, E, k):
    check(logits(T, E, dtype, T + k), k, dloss=2.0)
    check(tie_heavy_scores(T, E, dtype, 7), k, mask=torch.arange(T) % 5 != 1)
