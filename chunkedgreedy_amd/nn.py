"""Differentiable forms of the training operators, and the optimiser that uses
the orthogonalisation.

``embedding`` and ``layer_norm`` are ``sporder.embedding`` and
``sporder.layer_norm`` with their gradients behind torch's autograd; ``Muon``
updates weight matrices along the orthogonalised momentum
(``sporder.newton_schulz``).  Their backward passes are not differentiable in
turn, and they take neither forward-mode derivatives nor ``torch.func``'s
transforms (RuntimeError).  The end-to-end GCN (``e2e_gcn``) trains with them
on request.  They have no counterpart in the reference.
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
