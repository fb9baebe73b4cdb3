"""Linear with bias, activation and residual in its epilogue, and its gradients (not an ONNX node: a model that is
being exported calls ``linear`` and the operators of its own that the reference has for the rest)."""
import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .Checkpoint8 import _pack, _rows


def _dense(t):
    """Contiguous and at a multiple of 16 bytes, as the products load it."""
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


class LinearEpilogue(torch.autograd.Function):
    @staticmethod
    def forward(ctx, X, W, B, residual, in_features, out_features, activation, checkpoint8, train):
        name = "linear_epilogue"
        dev = _lib.require_gpu(name, X, W, B, residual)
        if activation not in _lib.ACTIVATIONS:
            raise ValueError("{}: activation must be one of {}, not {!r}".format(name, ", ".join(_lib.ACTIVATIONS),
                                                                               activation))
        act = _lib.ACTIVATIONS[activation]
        if tuple(W.shape) != (out_features, in_features):
            raise ValueError("{}: W {} does not match [out_features, in_features] = [{}, {}]".format(
                name, tuple(W.shape), out_features, in_features))
        N, K = W.shape
        if X.dim() == 0 or X.shape[-1] != K:
            raise ValueError("{}: X {} does not have W's {} features".format(name, tuple(X.shape), K))
        if activation == "swiglu" and N % 2:
            raise ValueError("{}: swiglu needs an even number of output features".format(name))
        lead, M = tuple(X.shape[:-1]), N // 2 if activation == "swiglu" else N
        if B is not None and tuple(B.shape) != (N,):
            raise ValueError("{}: B must be [out_features]".format(name))
        if residual is not None and tuple(residual.shape) != lead + (M,):
            raise ValueError("{}: residual must have the output's shape {}".format(name, lead + (M,)))
        if any(t is not None and t.dtype != W.dtype for t in (X, B, residual)):
            raise TypeError("{}: X, W, B and residual must share one dtype".format(name))
        dt = _lib.dtype_id(W, name)
        T = _rows(lead)
        need = ctx.needs_input_grad if train else (False,) * 4
        keep_h = activation != "none" and any(need[:3])
        L = _lib.lib()
        with _lib.on_device(dev):
            Xc, Wc = _dense(X), _dense(W)           # (autograd records nothing in here)
            Bc = None if B is None else B.contiguous()
            Rc = None if residual is None else residual.contiguous()
            Y = torch.empty(*lead, M, dtype=W.dtype, device=dev)
            H = torch.empty(L.opmx_linear_epilogue_kept_bytes(T, N, dt), dtype=torch.uint8, device=dev) if keep_h else None
            nbytes = L.opmx_linear_epilogue_workspace_bytes(T, K, N, dt, act)
            ws = _lib.workspace(nbytes, dev) if nbytes > 256 else None
            _lib.check(L.opmx_linear_epilogue(_lib.ptr(Xc), _lib.ptr(Wc), _lib.ptr(Bc), _lib.ptr(Rc), T, K, N, dt, act,
                                              _lib.ptr(Y), _lib.ptr(H), _lib.ptr(ws), nbytes if ws is not None else 0,
                                              _lib.stream_ptr(dev)), name)
            q = code = None
            if need[1] and checkpoint8:
                q, code = _pack(Xc, T, K, dev)
        if any(need[:3]):
            # inputs that were taken as they are get saved as themselves, so that autograd notices a change in place
            ctx.save_for_backward((X if Xc.data_ptr() == X.data_ptr() else Xc) if need[1] and not checkpoint8 else None,
                                  (W if Wc.data_ptr() == W.data_ptr() else Wc) if need[0] else None, H, q, code)
            ctx.sizes = (T, K, N, dt, act)
            ctx.shapes = (tuple(X.shape), W.dtype, dev)
        return Y

    @staticmethod
    @once_differentiable
    def backward(ctx, dY):
        need = ctx.needs_input_grad
        if not any(need[:3]):
            return None, None, None, dY, None, None, None, None, None
        X, W, H, q, code = ctx.saved_tensors
        T, K, N, dt, act = ctx.sizes
        xshape, dtype, dev = ctx.shapes
        L = _lib.lib()
        with _lib.on_device(dev):
            dYc = _dense(dY)
            dX = torch.empty(xshape, dtype=dtype, device=dev) if need[0] else None
            dW = torch.empty(N, K, dtype=dtype, device=dev) if need[1] else None
            dB = torch.empty(N, dtype=dtype, device=dev) if need[2] else None
            wanted = (_lib.LINEAR_DX * need[0] | _lib.LINEAR_DW * need[1] | _lib.LINEAR_DB * need[2]
                      | _lib.LINEAR_X8 * (q is not None))
            nbytes = L.opmx_linear_epilogue_gradients_workspace_bytes(T, K, N, dt, act, wanted)
            ws = _lib.workspace(nbytes, dev) if nbytes > 256 else None
            _lib.check(L.opmx_linear_epilogue_gradients(
                _lib.ptr(dYc), _lib.ptr(X), _lib.ptr(q), _lib.ptr(code), _lib.ptr(W), _lib.ptr(H), T, K, N, dt, act,
                _lib.ptr(dX), _lib.ptr(dW), _lib.ptr(dB), _lib.ptr(ws), nbytes if ws is not None else 0, _lib.stream_ptr(dev)),
                "linear_epilogue backward")
        return dX, dW, dB, dY if need[3] else None, None, None, None, None, None


def linear_epilogue(X: torch.Tensor, W: torch.Tensor, B: torch.Tensor, residual: torch.Tensor, in_features: int,
                    out_features: int, activation: str = "none", checkpoint8: bool = False):
    """``act(X W^T + B) + residual`` in one product: sums and epilogue in fp32, one rounding.

    X [*, in_features], W [out_features, in_features], B [out_features] or None; ``activation`` is none, silu, gelu,
    gelu_tanh or swiglu (as ``swiglu``: first half the gated one, output and residual [*, out_features / 2]).
    Differentiable in X, W, B and residual.  Where an activation needs it, X W^T + B is kept for the backward pass, in
    4 bytes per value for float32 and in 3 for the 16-bit types (under ``torch.no_grad`` nothing is).  For the gradients of X and W
    the gradient of X W^T + B is rounded to the tensors' type, as the matrix units take it: in float16 one past 65504 becomes an
    infinity there.  X, W and the gradient of the output are copied first where they are not contiguous or do not start at
    a multiple of 16 bytes.  ``checkpoint8``
    keeps X for the gradient of W in 8 bits (``checkpoint8_pack``) instead of as it is; the other gradients do not
    change.
    A backward pass is captured into a graph together with its forward pass, with no eager pass over the same leaves
    still alive: torch runs a backward pass on its forward pass's stream, which is not being captured."""
    return LinearEpilogue.apply(X, W, B, residual, in_features, out_features, activation, bool(checkpoint8),
                                torch.is_grad_enabled())
