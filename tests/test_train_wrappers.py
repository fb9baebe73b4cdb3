"""CPU: what the training operators refuse, in the package and at the C interface, before anything runs on a device."""
import ctypes

import pytest
import torch

import torch_function as OPMX
from torch_function import _lib

ONE = ctypes.c_void_p(256)      # never dereferenced on these paths


def test_no_cpu_path():
    x = torch.randn(4, 16)
    for call in (lambda: OPMX.checkpoint8_pack(x), lambda: OPMX.swiglu_checkpoint8(x),
                 lambda: OPMX.checkpoint8_unpack(torch.zeros(4, 16, dtype=torch.int8),
                                                 torch.zeros(4, 1, dtype=torch.uint8), torch.float32),
                 lambda: OPMX.moe_balance_loss(x, 16, 2),
                 lambda: OPMX.linear_epilogue(x, torch.randn(8, 16), None, None, 16, 8)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_public_names_and_signatures():
    import inspect
    sig = lambda f: list(inspect.signature(f).parameters)
    assert sig(OPMX.swiglu_checkpoint8) == ["X", "beta"]
    assert sig(OPMX.checkpoint8_pack) == ["X"] and sig(OPMX.checkpoint8_unpack) == ["q", "code", "dtype"]
    assert sig(OPMX.linear_epilogue) == ["X", "W", "B", "residual", "in_features", "out_features", "activation",
                                         "checkpoint8"]
    assert sig(OPMX.moe_balance_loss) == ["scores", "num_experts", "num_experts_per_token", "token_mask"]


def test_checkpoint8_c_interface():
    L = _lib.lib()
    assert L.opmx_checkpoint8_pack(ONE, -1, 8, 1, ONE, ONE, None) == -1
    assert L.opmx_checkpoint8_pack(ONE, 4, 8, 7, ONE, ONE, None) == -2
    for i in (0, 4, 5):
        a = [ONE, 4, 8, 1, ONE, ONE, None]
        a[i] = None
        assert L.opmx_checkpoint8_pack(*a) == -1
    assert L.opmx_checkpoint8_pack(None, 0, 8, 1, None, None, None) == 0
    assert L.opmx_checkpoint8_unpack(ONE, ONE, 4, -8, 1, ONE, None) == -1
    assert L.opmx_checkpoint8_unpack(ONE, ONE, 4, 8, 3, ONE, None) == -2
    assert L.opmx_checkpoint8_unpack(ONE, None, 4, 8, 1, ONE, None) == -1
    assert L.opmx_checkpoint8_unpack(None, None, 4, 0, 1, None, None) == 0
    assert L.opmx_swiglu_checkpoint8(ONE, 4, 8, 1.0, 9, ONE, ONE, ONE, None) == -2
    for i in (0, 5, 6, 7):
        a = [ONE, 4, 8, 1.0, 1, ONE, ONE, ONE, None]
        a[i] = None
        assert L.opmx_swiglu_checkpoint8(*a) == -1
    assert L.opmx_swiglu_checkpoint8(None, 0, 8, 1.0, 1, None, None, None, None) == 0
    for i in (0, 1, 2, 7):
        a = [ONE, ONE, ONE, 4, 8, 1.0, 1, ONE, None]
        a[i] = None
        assert L.opmx_swiglu_checkpoint8_backward(*a) == -1
    assert L.opmx_swiglu_checkpoint8_backward(ONE, ONE, ONE, 4, 8, 1.0, -1, ONE, None) == -2
    assert L.opmx_swiglu_checkpoint8_backward(None, None, None, 4, 0, 1.0, 1, None, None) == 0


def test_balance_loss_c_interface():
    L = _lib.lib()
    need = L.opmx_moe_balance_loss_workspace_bytes(4096, 64)
    assert need % 256 == 0 and need >= 256

    def call(scores=ONE, mask=None, T=4096, E=64, k=8, dtype=1, loss=ONE, count=ONE, w=ONE, ws=ONE, bytes_=need):
        return L.opmx_moe_balance_loss(scores, mask, T, E, k, dtype, loss, count, w, ws, bytes_, None)

    assert call(T=-1) == -1 and call(E=0) == -1 and call(k=0) == -1 and call(k=65) == -1
    assert call(E=257) == -2 and call(k=33) == -2 and call(dtype=4) == -2 and call(T=1 << 40) == -2
    assert call(scores=None) == -1 and call(loss=None) == -1 and call(count=None) == -1 and call(w=None) == -1
    assert call(ws=None) == -3 and call(bytes_=need - 1) == -3 and call(ws=ctypes.c_void_p(264)) == -4

    def back(scores=ONE, w=ONE, d=ONE, T=8, E=8, dtype=1, out=ONE):
        return L.opmx_moe_balance_loss_backward(scores, None, w, d, T, E, dtype, out, None)

    assert back(T=-1) == -1 and back(E=0) == -1 and back(E=300) == -2 and back(dtype=9) == -2
    assert back(scores=None) == -1 and back(w=None) == -1 and back(d=None) == -1 and back(out=None) == -1
    assert back(None, None, None, 0, 8, 1, None) == 0


def test_linear_epilogue_c_interface():
    L = _lib.lib()
    odd = ctypes.c_void_p(258)
    need = L.opmx_linear_epilogue_workspace_bytes(100, 4000, 512, 1, 0)
    assert need % 256 == 0 and need > 256            # cut along k

    def call(X=ONE, W=ONE, T=100, K=4000, N=512, dtype=1, act=0, Y=ONE, ws=ONE, bytes_=need):
        return L.opmx_linear_epilogue(X, W, None, None, T, K, N, dtype, act, Y, None, ws, bytes_, None)

    assert call(T=-1) == -1 and call(K=-1) == -1 and call(K=0) == -1 and call(act=5) == -1 and call(act=-1) == -1
    assert call(N=511, act=4) == -1 and call(X=None) == -1 and call(W=None) == -1 and call(Y=None) == -1
    assert call(dtype=3) == -2 and call(K=1 << 21) == -2 and call(N=1 << 21) == -2 and call(T=1 << 31) == -2
    assert call(X=odd) == -4 and call(W=odd) == -4 and call(ws=ctypes.c_void_p(128)) == -4
    assert call(ws=None) == -3 and call(bytes_=need - 1) == -3
    assert call(None, None, 0, 4000, 512, 1, 0, None, None, 0) == 0
    need = L.opmx_linear_epilogue_backward_workspace_bytes(64, 4000, 512, 1, 1)

    def back(dY=ONE, X=ONE, q=None, code=None, W=ONE, H=ONE, T=64, K=4000, N=512, dtype=1, act=1, dX=ONE, dW=ONE, dB=ONE,
             ws=ONE, bytes_=need):
        return L.opmx_linear_epilogue_backward(dY, X, q, code, W, H, T, K, N, dtype, act, dX, dW, dB, ws, bytes_, None)

    assert back(T=-1) == -1 and back(K=0) == -1 and back(N=0) == -1 and back(act=9) == -1 and back(N=511, act=4) == -1
    assert back(dtype=9) == -2 and back(K=1 << 21) == -2
    assert back(dY=None) == -1 and back(H=None) == -1 and back(W=None) == -1 and back(X=None) == -1
    assert back(q=ONE) == -1 and back(code=ONE) == -1 and back(X=None, q=ONE) == -1
    assert back(X=odd) == -4 and back(W=odd) == -4 and back(dY=odd, act=0) == -4
    assert back(H=ctypes.c_void_p(264)) == -4
    assert L.opmx_linear_epilogue_kept_bytes(5, 7, 1) == 105 and L.opmx_linear_epilogue_kept_bytes(5, 7, 0) == 140
    assert back(ws=None) == -3 and back(bytes_=need - 1) == -3 and back(ws=ctypes.c_void_p(257)) == -4
    assert back(dX=None, dW=None, dB=None) == 0


@pytest.mark.gpu
def test_package_refusals():
    d = torch.device("cuda:0")
    x = torch.randn(4, 15, device=d)
    with pytest.raises(ValueError, match="even"):
        OPMX.swiglu_checkpoint8(x)
    with pytest.raises(TypeError):
        OPMX.swiglu_checkpoint8(x[:, :14].double())
    with pytest.raises(TypeError):
        OPMX.checkpoint8_pack(x.int())
    q, code = OPMX.checkpoint8_pack(x)
    with pytest.raises(TypeError):
        OPMX.checkpoint8_unpack(q.int(), code, torch.float32)
    with pytest.raises(TypeError):
        OPMX.checkpoint8_unpack(q, code, torch.int32)
    with pytest.raises(ValueError):
        OPMX.checkpoint8_unpack(q, code[:3], torch.float32)
    for a in ((x, 8, 2), (x, 15, 0), (x, 15, 16), (x, 15, 2, torch.ones(4, device=d)),
              (x, 15, 2, torch.ones(3, dtype=torch.bool, device=d))):
        with pytest.raises(ValueError):
            OPMX.moe_balance_loss(*a)
    with pytest.raises(TypeError):
        OPMX.moe_balance_loss(x.double(), 15, 2)
    with pytest.raises(RuntimeError, match="no CPU path"):
        OPMX.moe_balance_loss(x, 15, 2, torch.ones(4, dtype=torch.bool))
    W, lin = torch.randn(6, 15, device=d), OPMX.linear_epilogue
    for a in ((x, W, None, None, 14, 6), (x, W, None, None, 15, 5), (x[:, :14], W, None, None, 15, 6),
              (x, W, W[0], None, 15, 6), (x, W, None, x, 15, 6), (x, W, None, None, 15, 6, "relu"),
              (x, W[:5], None, None, 15, 5, "swiglu"), (x, W, None, torch.zeros(6, device=d), 15, 6)):
        with pytest.raises(ValueError):
            lin(*a)
    for a in ((x.half(), W, None, None, 15, 6), (x, W, W[:, 0].half().contiguous(), None, 15, 6),
              (x.double(), W.double(), None, None, 15, 6)):
        with pytest.raises(TypeError):
            lin(*a)
    leaf = x[:, :14].clone().requires_grad_(True)
    y = OPMX.swiglu_checkpoint8(leaf)
    g, = torch.autograd.grad(y, leaf, torch.ones_like(y).requires_grad_(True), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


def test_swiglu_checkpoint8_keeps_both_or_nothing():
    L = _lib.lib()
    assert L.opmx_swiglu_checkpoint8(ONE, 4, 8, 1.0, 1, ONE, ONE, None, None) == -1
    assert L.opmx_swiglu_checkpoint8(ONE, 4, 8, 1.0, 1, ONE, None, ONE, None) == -1
    assert L.opmx_swiglu_checkpoint8(ONE, 0, 8, 1.0, 1, ONE, None, None, None) == 0


def test_balance_loss_refuses_counts_past_32_bits():
    """2^31 tokens in all would be -2^31 in the sums on the way."""
    L = _lib.lib()
    T = 1 << 31
    for k, first in ((1, T), (2, T // 2), (8, T // 8), (7, T // 7 + 1)):
        need = L.opmx_moe_balance_loss_workspace_bytes(first, 8)
        assert L.opmx_moe_balance_loss(ONE, None, first, 8, k, 1, ONE, ONE, ONE, ONE, need, None) == -2
        assert L.opmx_moe_balance_loss(ONE, None, first - 1, 8, k, 1, ONE, ONE, ONE, ONE, need - 1, None) == -3


def test_balance_loss_workspace_holds_every_block():
    """A block's sums are 8 bytes an expert (rows of four) and 4; more than 8 picks take 16 tokens a block at a time (64 up to 64
    experts), so that 4096 tokens of 100 experts fill 256 blocks."""
    L = _lib.lib()
    for T, E, blocks in ((4096, 100, 256), (200, 100, 13), (1 << 20, 256, 256), (4096, 16, 64), (8192, 64, 256)):
        assert L.opmx_moe_balance_loss_workspace_bytes(T, E) >= blocks * ((E + 3) // 4 * 32 + 4)
    assert L.opmx_moe_balance_loss_workspace_bytes(64, 256) == 256 == L.opmx_moe_balance_loss_workspace_bytes(32, 8)


def test_gradients_ask_for_what_they_need():
    """The workspace holds dH, where it is not dY; X where it is padded or unpacked; W where it is padded; the sums for dB; the
    sums of k ranges: each only where a wanted gradient takes it."""
    L = _lib.lib()
    up = lambda v: -(-v // 256) * 256
    DX, DW, DB, X8 = 1, 2, 4, 8
    T, K, N, bf = 8192, 14336, 4096, 2
    need = lambda act, wanted, T=T, K=K, N=N, dt=bf: L.opmx_linear_epilogue_gradients_workspace_bytes(T, K, N, dt, act, wanted)
    assert need(0, DX) == need(0, DW) == need(0, DX | DW) == 256                     # many rows: no k ranges
    assert need(0, DX | X8) == 256 and need(0, DW | X8) == up(T * K * 2)
    assert need(1, DX) == need(1, DX | DW) == up(T * N * 2)
    sums = need(0, DB)
    assert 256 < sums <= up(512 * N * 4) and need(1, DB) == sums
    assert need(1, DX | DW | DB | X8) == up(T * N * 2) + up(T * K * 2) + sums
    odd = dict(T=900, K=4001, N=3999)                                               # pitches 4008 and 4000
    w, x, dh = up(3999 * 4008 * 2), up(900 * 4008 * 2), up(900 * 4000 * 2)
    assert dh + w <= need(1, DX, **odd) < dh + w + x
    assert dh + x <= need(1, DW, **odd) < dh + w + x
    assert need(1, DB, **odd) < dh
    assert need(0, DX | DW | DB, T=0, K=4001, N=4096) == L.opmx_linear_epilogue_gradients_workspace_bytes(0, 4001, 4096, bf, 0, DW | DB)
    any_ = L.opmx_linear_epilogue_backward_workspace_bytes
    for case in ((8192, 14336, 4096, bf, 0), (900, 4001, 3999, 1, 4), (64, 4000, 512, 0, 1), (5, 33, 7, 0, 2), (0, 40, 8, 1, 3)):
        sizes = [L.opmx_linear_epilogue_gradients_workspace_bytes(*case, w) for w in range(16)]
        assert max(sizes) == any_(*case)
    # the call takes exactly that, and the older entry point what may be asked for at most
    size = need(1, DW, T=64, K=4000, N=512, dt=1)
    a = [ONE, ONE, None, None, ONE, ONE, 64, 4000, 512, 1, 1, None, ONE, None, ONE]
    assert L.opmx_linear_epilogue_gradients(*a, size - 1, None) == -3
    assert L.opmx_linear_epilogue_backward(*a, size, None) == -3
    a[1], a[2], a[3] = None, ONE, ONE
    assert L.opmx_linear_epilogue_gradients(*a, size, None) == -3


def test_a_workspace_that_is_needed_is_not_called_none():
    """256 bytes mean that there may be no workspace: the smallest dH, the smallest sums for dB and the smallest padded operand,
    of 256 bytes and less, are more than that, and without a workspace the call is refused."""
    L = _lib.lib()
    DX, DW, DB, X8 = 1, 2, 4, 8
    for T, K, N, dt, act, wanted in ((1, 64, 64, 1, 0, DB), (1, 64, 64, 1, 0, DX | DW | DB), (3, 100, 36, 0, 0, DB), (1, 64, 64, 1, 1, DX),
                                     (1, 8, 8, 1, 0, DW | X8), (1, 1, 8, 2, 0, DX), (1, 1, 8, 2, 0, DW), (1, 1, 1, 0, 4, DW)):
        need = L.opmx_linear_epilogue_gradients_workspace_bytes(T, K, N, dt, act, wanted)
        assert need >= 512, (T, K, N, dt, act, wanted)
        if act == 4:
            continue
        out = [ONE if wanted & bit else None for bit in (DX, DW, DB)]
        x8 = ONE if wanted & X8 else None
        for ws, size in ((None, 0), (None, need), (ONE, need - 1), (ONE, 256)):
            assert L.opmx_linear_epilogue_gradients(ONE, ONE, x8, x8, ONE, ONE, T, K, N, dt, act, *out, ws, size, None) == -3
    for T in (0, 1, 17, 33, 65, 130, 1000):
        for K, N in ((8, 8), (64, 16), (1000, 24), (8192, 64)):
            for act in range(5):
                for dt in range(3):
                    plain = L.opmx_linear_epilogue_gradients_workspace_bytes(T, K, N, dt, act, DB)
                    assert plain >= 512 if T else plain == 256


def test_the_quicker_kernel_for_few_rows():
    """The kernels for few rows need no workspace.  The tile product needs one where it copies rows that are no whole chunks, or
    cuts k.  Each size with the microseconds of the kernels for few rows and of the tile product."""
    L = _lib.lib()
    tiles = [(16, 14335, 128, 1, 0), (8, 14335, 1024, 1, 0), (32, 14335, 1024, 1, 0), (32, 4095, 1024, 1, 0), (20, 8191, 512, 1, 4),
             (32, 4096, 1024, 1, 0), (20, 4096, 1024, 0, 0), (8, 14336, 128, 1, 0), (64, 14335, 4096, 1, 0), (64, 1001, 28672, 1, 0),
             (32, 1001, 28672, 2, 0)]    # 88 17, 73 30, 131 30, 40 17, 87 24, 14 10, 25 14, 35 17, 153 54, 80 39, 57 39
    few = [(64, 501, 4096, 0, 0), (40, 250, 1024, 1, 0), (16, 1001, 4096, 1, 0), (4, 4095, 14336, 0, 0), (32, 4095, 4096, 0, 0),
           (1, 4096, 28672, 1, 4), (16, 4096, 4096, 2, 0), (20, 1024, 4096, 1, 0), (64, 512, 2816, 1, 0), (64, 1024, 2816, 0, 2)]
    #      9.6 17, 3.8 7.2, 7.8 17, 73 151, 37 48, 38 50, 9 14, 5.4 9.0, 5.5 6.7, 13.0 12.8
    for case in tiles:
        assert L.opmx_linear_epilogue_workspace_bytes(*case) > 256, case
    for case in few:
        assert L.opmx_linear_epilogue_workspace_bytes(*case) == 256, case
