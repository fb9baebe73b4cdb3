"""Activations kept in 8 bits for the backward pass, and SwiGLU that keeps its input so (no counterpart in
the reference, which only runs forward; not ONNX nodes).

Blocks of 32 values of the last dimension share a power-of-two step and hold whole numbers in [-127, 127]:
8.25 bits per value instead of 16 or 32, off by at most 1/127.5 of the block's largest magnitude or 2^-127, whichever is
more (``include/opmx_moe.h`` has the definition).  A block with an infinity or a NaN stands for NaN throughout.
"""
import torch
from torch.autograd.function import once_differentiable

from . import _lib

BLOCK = 32


def _blocks(D):
    return (D + BLOCK - 1) // BLOCK


def _pack(X, R, D, dev):
    """q int8 [R, D] and code uint8 [R, ceil(D/32)] of the contiguous rows of X."""
    q = torch.empty(R, D, dtype=torch.int8, device=dev)
    code = torch.empty(R, _blocks(D), dtype=torch.uint8, device=dev)
    _lib.check(_lib.lib().opmx_checkpoint8_pack(_lib.ptr(X), R, D, _lib.dtype_id(X, "checkpoint8_pack"), _lib.ptr(q),
                                                _lib.ptr(code), _lib.stream_ptr(dev)), "checkpoint8_pack")
    return q, code


def checkpoint8_pack(X: torch.Tensor):
    """-> (q int8 [*, D], code uint8 [*, ceil(D/32)]): X in 8 bits.  Not differentiable."""
    dev = _lib.require_gpu("checkpoint8_pack", X)
    if X.dim() == 0:
        raise ValueError("checkpoint8_pack: X needs at least one dimension")
    _lib.dtype_id(X, "checkpoint8_pack")
    lead, D = tuple(X.shape[:-1]), X.shape[-1]
    with _lib.on_device(dev):
        Xc = X.detach().contiguous()
        q, code = _pack(Xc, _rows(lead), D, dev)
    return q.view(*lead, D), code.view(*lead, _blocks(D))


def checkpoint8_unpack(q: torch.Tensor, code: torch.Tensor, dtype: torch.dtype):
    """The values that ``checkpoint8_pack``'s result stands for, as a tensor of ``dtype``."""
    dev = _lib.require_gpu("checkpoint8_unpack", q, code)
    if q.dtype != torch.int8 or code.dtype != torch.uint8:
        raise TypeError("checkpoint8_unpack: q must be int8 and code uint8")
    if q.dim() == 0 or tuple(code.shape) != tuple(q.shape[:-1]) + (_blocks(q.shape[-1]),):
        raise ValueError("checkpoint8_unpack: code must be [*, ceil(D/32)] for q [*, D]")
    lead, D = tuple(q.shape[:-1]), q.shape[-1]
    with _lib.on_device(dev):
        X = torch.empty(*lead, D, dtype=dtype, device=dev)
        qc, cc = q.contiguous(), code.contiguous()
        _lib.check(_lib.lib().opmx_checkpoint8_unpack(_lib.ptr(qc), _lib.ptr(cc), _rows(lead), D,
                                                      _lib.dtype_id(X, "checkpoint8_unpack"), _lib.ptr(X),
                                                      _lib.stream_ptr(dev)), "checkpoint8_unpack")
    return X


def _rows(lead):
    n = 1
    for s in lead:
        n *= s
    return n


class SwiGLUCheckpoint8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, X, beta, train):
        dev = _lib.require_gpu("swiglu_checkpoint8", X)
        if X.dim() == 0 or X.shape[-1] % 2:
            raise ValueError("swiglu_checkpoint8: last dimension must be even")
        dt = _lib.dtype_id(X, "swiglu_checkpoint8")
        lead, D = tuple(X.shape[:-1]), X.shape[-1] // 2
        R = _rows(lead)
        # (ctx.needs_input_grad tells what X asks for, also where nothing is recorded)
        keep = train and ctx.needs_input_grad[0]
        with _lib.on_device(dev):
            Xc = X.detach().contiguous()
            Y = torch.empty(*lead, D, dtype=X.dtype, device=dev)
            q = torch.empty(R, 2, D, dtype=torch.int8, device=dev) if keep else None
            code = torch.empty(R, 2, _blocks(D), dtype=torch.uint8, device=dev) if keep else None
            _lib.check(_lib.lib().opmx_swiglu_checkpoint8(_lib.ptr(Xc), R, D, float(beta), dt, _lib.ptr(Y), _lib.ptr(q),
                                                          _lib.ptr(code), _lib.stream_ptr(dev)), "swiglu_checkpoint8")
        if keep:
            ctx.save_for_backward(q, code)
            ctx.beta, ctx.dtype, ctx.shape = float(beta), X.dtype, tuple(X.shape)
        return Y

    @staticmethod
    @once_differentiable
    def backward(ctx, dY):
        q, code = ctx.saved_tensors
        dev, D = q.device, q.shape[-1]
        with _lib.on_device(dev):
            dYc = dY.contiguous()
            dX = torch.empty(ctx.shape, dtype=ctx.dtype, device=dev)
            _lib.check(_lib.lib().opmx_swiglu_checkpoint8_backward(
                _lib.ptr(dYc), _lib.ptr(q), _lib.ptr(code), q.shape[0], D, ctx.beta,
                _lib.dtype_id(dX, "swiglu_checkpoint8"), _lib.ptr(dX), _lib.stream_ptr(dev)), "swiglu_checkpoint8")
        return dX, None, None


def swiglu_checkpoint8(X: torch.Tensor, beta: float = 1.0):
    """``swiglu`` for training: the same output (and finite also where the product of the halves alone is beyond fp32, which
    ``swiglu`` makes an infinity or a NaN), and the gradient of X taken at X as 8 bits hold it.  Where no gradient is asked for, or
    under ``torch.no_grad``, nothing is kept.  X may be changed in place afterwards: only its 8-bit form is used."""
    return SwiGLUCheckpoint8.apply(X, beta, torch.is_grad_enabled())
