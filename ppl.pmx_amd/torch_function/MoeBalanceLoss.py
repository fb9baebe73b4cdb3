"""Balance loss of the router with the tokens per expert (no counterpart in the reference, whose router only
runs forward; not an ONNX node)."""
import torch
from torch.autograd.function import once_differentiable

from . import _lib


class MoeBalanceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, scores, num_experts, num_experts_per_token, token_mask):
        E, k = int(num_experts), int(num_experts_per_token)
        dev = _lib.require_gpu("moe_balance_loss", scores, token_mask)
        if scores.dim() == 0 or scores.shape[-1] != E:
            raise ValueError("moe_balance_loss: scores shape {} does not match num_experts {}".format(
                tuple(scores.shape), E))
        if not (1 <= k <= E):
            raise ValueError("moe_balance_loss: need 1 <= num_experts_per_token <= num_experts")
        if token_mask is not None and (token_mask.dtype != torch.bool or token_mask.shape != scores.shape[:-1]):
            raise ValueError("moe_balance_loss: token_mask must be a bool tensor of the shape of scores without its "
                             "last dimension")
        dt = _lib.dtype_id(scores, "moe_balance_loss")
        T = scores.numel() // E
        L = _lib.lib()
        with _lib.on_device(dev):
            sc = scores.detach().contiguous()
            mc = None if token_mask is None else token_mask.contiguous()
            loss = torch.empty((), dtype=torch.float32, device=dev)
            count = torch.empty(E, dtype=torch.int64, device=dev)
            weight = torch.empty(E, dtype=torch.float32, device=dev)
            nbytes = L.opmx_moe_balance_loss_workspace_bytes(T, E)
            ws = _lib.workspace(nbytes, dev) if nbytes > 256 else None
            _lib.check(L.opmx_moe_balance_loss(_lib.ptr(sc), _lib.ptr(mc), T, E, k, dt, _lib.ptr(loss), _lib.ptr(count),
                                               _lib.ptr(weight), _lib.ptr(ws), nbytes, _lib.stream_ptr(dev)),
                       "moe_balance_loss")
        if ctx.needs_input_grad[0]:
            # a contiguous input is saved as itself, so autograd notices a change in place before the backward pass
            own = scores.is_contiguous()
            ctx.save_for_backward(scores if own else sc, token_mask if mc is token_mask else mc, weight)
            ctx.E = E
        ctx.mark_non_differentiable(count)
        return loss, count

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, _):
        scores, mask, weight = ctx.saved_tensors
        dev, E = scores.device, ctx.E
        with _lib.on_device(dev):
            d = dloss.to(torch.float32).contiguous()
            ds = torch.empty_like(scores, memory_format=torch.contiguous_format)
            _lib.check(_lib.lib().opmx_moe_balance_loss_backward(
                _lib.ptr(scores), _lib.ptr(mask), _lib.ptr(weight), _lib.ptr(d), scores.numel() // E, E,
                _lib.dtype_id(scores, "moe_balance_loss"), _lib.ptr(ds), _lib.stream_ptr(dev)), "moe_balance_loss")
        return ds, None, None, None


def moe_balance_loss(scores: torch.Tensor, num_experts: int, num_experts_per_token: int, token_mask: torch.Tensor = None):
    """-> (loss, expert_count [E] i64) of the router logits ``scores`` [*, E].

    With p the softmax of a token's scores, count[e] the tokens that pick expert e (the picks of ``moe_select``:
    differences of its expert_offset), n the number of tokens and f = count / (k n):
    ``loss = E * sum_e f_e * mean_t p[t, e]``, a float32 scalar, 1 for a router that spreads evenly.  The gradient
    reaches ``scores`` through p; f is held constant.  ``token_mask`` (bool [*]): tokens that are False, padding for
    instance, count nowhere and get a zero gradient."""
    return MoeBalanceLoss.apply(scores, num_experts, num_experts_per_token, token_mask)
