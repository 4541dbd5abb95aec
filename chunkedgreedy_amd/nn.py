"""Differentiable forms of the training operators, and the optimiser that uses
the orthogonalisation.

``embedding``, ``layer_norm``, ``dropout``, ``residual_norm`` and
``linear_cross_entropy`` are ``sporder``'s with their gradients behind torch's
autograd; ``Dropout`` holds a seed and counts its calls; ``Muon`` updates weight
matrices along the orthogonalised momentum (``sporder.newton_schulz``).  Their
backward passes are not differentiable in turn, and they take neither
forward-mode derivatives nor ``torch.func``'s transforms (RuntimeError).  The
end-to-end GCN (``e2e_gcn``) trains with them on request.  They have no
counterpart in the reference.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import sporder
from .sporder import _train


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, tokens, scale, padding_idx):
        ctx.save_for_backward(tokens)
        out = sporder.embedding(table, tokens, scale=scale)
        _train._padding_row(padding_idx, table.shape[0])  # the table has passed its own checks
        ctx.rows, ctx.scale, ctx.padding_idx = table.shape[0], scale, padding_idx
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        (tokens,) = ctx.saved_tensors
        return sporder.embedding_grad(grad, tokens, ctx.rows, scale=ctx.scale,
                                      padding_idx=ctx.padding_idx), None, None, None


def embedding(table, tokens, *, scale=1.0, padding_idx=None):
    """scale * table[tokens]; the table's gradient is dense, and zero for the
    row ``padding_idx`` (if given) and for rows without a token."""
    return _Embedding.apply(table, tokens, scale, padding_idx)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = sporder.layer_norm(x, weight, bias, eps=eps)
        ctx.save_for_backward(x, mean, rstd, weight)
        ctx.bias_type = None if bias is None else bias.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, mean, rstd, weight = ctx.saved_tensors
        dx, dweight, dbias = sporder.layer_norm_grad(grad, x, mean, rstd, weight)
        return (dx, None if weight is None else dweight,
                None if ctx.bias_type is None else dbias.to(ctx.bias_type), None)


def layer_norm(x, weight=None, bias=None, *, eps=1e-5):
    """Layer norm of the last dimension, differentiable by x, weight and bias."""
    return _LayerNorm.apply(x, weight, bias, eps)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, offset):
        if isinstance(seed, torch.Tensor):
            seed = seed.clone()  # the backward pass needs what this call reads
            ctx.save_for_backward(seed)
        ctx.p, ctx.seed, ctx.offset = p, seed, offset
        return sporder.dropout(x, p, seed, offset=offset, residual=residual)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        (seed,) = ctx.saved_tensors or (ctx.seed,)
        dx = None
        if ctx.needs_input_grad[0]:
            dx = sporder.dropout(grad, ctx.p, seed, offset=ctx.offset)
        return dx, grad if ctx.needs_input_grad[1] else None, None, None, None


def dropout(x, p, seed, *, offset=0, residual=None, training=True):
    """residual + dropout of x, whose mask follows from seed and offset
    (``sporder.dropout``) and is made again for the gradient; x (plus residual)
    itself where not ``training``."""
    if not training:
        return x if residual is None else x + residual
    return _Dropout.apply(x, residual, p, seed, offset)


class Dropout(torch.nn.Module):
    """Dropout with its own seed and a count of its calls, held on the GPU so that
    each replay of a captured step drops other elements.  Modules of one model
    have different seeds, or they drop the same elements.  A part that is run again
    for its gradients needs ``dropout`` with an offset of its own instead: its
    second run would count on."""

    def __init__(self, p=0.5, seed=0):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError("p must be in [0, 1]")
        self.p = p
        if not -(2**63) <= seed < 2**64:
            raise ValueError("seed must be in [0, 2^64)")
        signed = seed - 2**64 if seed >= 2**63 else seed  # the same 64 bits
        self.register_buffer("state", torch.tensor([signed, 0], dtype=torch.int64))

    def forward(self, x, residual=None):
        out = dropout(x, self.p, self.state, residual=residual, training=self.training)
        if self.training:
            self.state[1] += 1
        return out


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, gate, post_weight, weight, scale, eps, post_norm):
        ctx.set_materialize_grads(False)
        y, h, post_rstd, rstd = sporder.residual_norm(x, residual, gate, post_weight, weight,
                                                      scale=scale, eps=eps, post_norm=post_norm)
        ctx.save_for_backward(x, y, post_rstd, rstd, gate, post_weight, weight)
        ctx.scale, ctx.post_norm = scale, post_norm
        return y, h

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y, grad_h):
        x, y, post_rstd, rstd, gate, post_weight, weight = ctx.saved_tensors
        dx, dresidual, dgate, dpost, dweight = sporder.residual_norm_grad(
            grad_y, grad_h, x, y, post_rstd, rstd, gate, post_weight, weight, scale=ctx.scale,
            post_norm=ctx.post_norm)
        return (dx, dresidual if ctx.needs_input_grad[1] else None, dgate, dpost, dweight,
                None, None, None)


def residual_norm(x, residual=None, gate=None, post_weight=None, weight=None, *, scale=1.0,
                  eps=1e-5, post_norm=True):
    """(y, h): the residual stream after a block and the next block's input
    (``sporder.residual_norm``), differentiable by all five tensors."""
    return _ResidualNorm.apply(x, residual, gate, post_weight, weight, scale, eps, post_norm)


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, targets, bias, ignore_index, reduction):
        loss, lse, sums = sporder.linear_cross_entropy(x, weight, targets, bias,
                                                       ignore_index=ignore_index)
        ctx.save_for_backward(x, weight, targets, bias, lse, sums, loss)
        ctx.ignore_index, ctx.reduction = ignore_index, reduction
        if reduction == "none":
            return loss.clone()  # the caller may write to it, and the backward pass reads this one
        return sums[0] / sums[1] if reduction == "mean" else sums[0].clone()

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, targets, bias, lse, sums, loss = ctx.saved_tensors
        if ctx.reduction == "mean":
            grad = grad / sums[1]
        dx, dweight, dbias = sporder.linear_cross_entropy_grad(
            grad, x, weight, targets, lse, bias, ignore_index=ctx.ignore_index, loss=loss)
        return dx, dweight, None, dbias, None, None


def linear_cross_entropy(x, weight, targets, bias=None, *, ignore_index=-100, reduction="mean"):
    """Softmax cross entropy of the logits x weight^T + bias, which are never kept
    (``sporder.linear_cross_entropy``), differentiable by x, weight and bias: the
    mean over the rows that are not ignored, their sum, or the losses by row."""
    if reduction not in ("mean", "sum", "none"):
        raise ValueError("reduction must be mean, sum or none")
    return _LinearCrossEntropy.apply(x, weight, targets, bias, ignore_index, reduction)


class Muon(torch.optim.Optimizer):
    """Momentum whose update is orthogonalised, for parameters of two (or, as a
    batch of matrices, three) dimensions:

        m <- momentum m + g
        W <- W - lr sqrt(max(1, rows / cols)) NewtonSchulz(g + momentum m)

    Each singular direction of the update moves the weight by about the same
    amount; the root keeps the update's mean square the same for tall matrices.
    The momentum and the update are float32 whatever the parameter's type, in
    whose 16 bits a sum of small gradients would be lost or pass the range; the
    parameter is rounded once a step.  Parameters without a gradient or without
    elements are passed over; a parameter that newton_schulz refuses ends the
    step (ValueError or TypeError) before any of them changes.
    """

    def __init__(self, params, lr=0.02, momentum=0.95, steps=5):
        if not lr >= 0.0 or not 0.0 <= momentum < 1.0:
            raise ValueError("lr must be >= 0 and momentum in [0, 1)")
        super().__init__(params, {"lr": lr, "momentum": momentum, "steps": steps})
        for group in self.param_groups:
            for p in group["params"]:
                if p.dim() not in (2, 3):
                    raise ValueError("Muon takes parameters of two or three dimensions, got "
                                     f"shape {tuple(p.shape)}")

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        # What can be refused is refused before any parameter or state changes.
        todo = [(p, group) for group in self.param_groups for p in group["params"]
                if p.grad is not None and p.numel() > 0]
        for p, group in todo:
            _train._step_count(group["steps"])
            if p.grad.layout != torch.strided:
                raise ValueError("Muon takes dense gradients")
            _train._matrices(p.grad, "a parameter's gradient")
        for p, group in todo:
            state = self.state[p]
            if "momentum" not in state:
                state["momentum"] = torch.zeros_like(p, dtype=torch.float32)
            m = state["momentum"]
            m.mul_(group["momentum"]).add_(p.grad)
            update = sporder.newton_schulz(p.grad.float().add(m, alpha=group["momentum"]),
                                           steps=group["steps"])
            p.add_(update, alpha=-group["lr"] * max(1.0, p.shape[-2] / p.shape[-1]) ** 0.5)
        return loss

    def load_state_dict(self, state_dict):
        """As torch's, which rounds the state to the parameters' types: the
        momentum is taken from ``state_dict`` in float32."""
        super().load_state_dict(state_dict)
        ids = (i for group in state_dict["param_groups"] for i in group["params"])
        params = (p for group in self.param_groups for p in group["params"])
        for i, p in zip(ids, params):
            held = state_dict["state"].get(i, {}).get("momentum")
            if held is not None:
                self.state[p]["momentum"] = held.to(device=p.device, dtype=torch.float32)
