"""``orthogonalize``: matrices with their singular values driven towards one, and ``Muon``, the optimiser that takes such updates.

The weights of a Pairformer stack are matrices, many of one shape (128 x 128, 512 x 128 and 128 x 512 in the pair path of each block, 384 x 384 to 1536 x
384 in the single one).  The stack of this package runs forward only and gives them no gradient: they are updated where other code trains them.  What the operators
of this package train are the matrices around them: projections, heads, the weight of the position encoding.

A momentum whose singular values are made alike moves all directions of a weight by the same amount.  The polynomial iteration (Newton-Schulz) needs products
only; ``px_orthogonalize`` runs it for all matrices of a shape at once.
"""
from __future__ import annotations

import math
from typing import Iterable, Optional, Sequence, Tuple, Union

import torch

from . import native

Coefficients = Union[Tuple[float, float, float], Sequence[Tuple[float, float, float]]]
DEFAULT = (3.4445, -4.7750, 2.0315)


def orthogonalize(g: torch.Tensor, steps: int = 5, coefficients: Coefficients = DEFAULT, eps: float = 1e-7) -> torch.Tensor:
    """Each matrix of ``g`` [..., M, N] with its singular values near one; a new tensor of g's shape and type (fp32, bf16 or fp16).

    X = g / (|g| + eps), |g| the root of the sum of squares, then ``steps`` times X <- a X + b (X X^T) X + c (X X^T)^2 X with (a, b, c) =
    ``coefficients``, or one triple for each step (``steps`` is then their number).  The default triple takes singular values above 0.01 |g| to
    between 0.7 and 1.2 in five steps.

    Products take operands of 22 bits and add in fp32 whatever the type: 16-bit iterates lose up to a third of the result where singular values differ
    much.  Iterates and polynomials of up to 60 are held; an overflow comes out infinite or NaN.  A matrix that is not finite gives NaN, a zero one zero (eps > 0).
    Up to 65535 matrices of 2^20 rows and columns.  Not differentiable: g is detached or no_grad is in force.
    """
    if not g.is_cuda:
        raise RuntimeError("orthogonalize: CUDA tensors only, this package has no CPU path")
    single = len(coefficients) > 0 and isinstance(coefficients[0], (int, float))
    triples = [tuple(coefficients)] * int(steps) if single else [tuple(c) for c in coefficients]
    if any(len(c) != 3 for c in triples):
        raise RuntimeError("orthogonalize: coefficients are triples (a, b, c)")
    return native.load().orthogonalize(g, [float(x) for c in triples for x in c], eps)


class Muon(torch.optim.Optimizer):
    """Momentum whose matrices are orthogonalised before they are applied.

    For each parameter p [..., M, N] with gradient g: buf <- momentum buf + g, u = g + momentum buf (``nesterov``) or buf,
    p <- (1 - lr weight_decay) p - lr sqrt(max(1, M / N)) orthogonalize(u).  Parameters of one shape and type are orthogonalised in one call.  For weights
    with two axes or more; biases, norms and tables of embeddings want another optimiser beside it.  fp32, bf16 and fp16 CUDA parameters, up to 65535 matrices
    of a shape and type; a step that is refused has changed nothing.

    The momentum is fp32 whatever the parameter's type, in checkpoints too, and u, its orthogonalisation and the new weight are formed in fp32 and rounded
    once, to the parameter.  What is below half a step of a 16-bit weight (2^-9 to 2^-8 of it in bf16), a small decay beside a small update for one, leaves no
    trace in it: keep the parameters in fp32 and round them for the forward pass where that matters.
    """

    def __init__(self, params: Iterable[torch.Tensor], lr: float = 0.02, momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0,
                 steps: int = 5, coefficients: Coefficients = DEFAULT, eps: float = 1e-7) -> None:
        if not lr >= 0.0 or not 0.0 <= momentum < 1.0 or not weight_decay >= 0.0:
            raise ValueError("Muon: lr and weight_decay must not be negative, momentum must lie in [0, 1)")
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps, coefficients=coefficients, eps=eps))

    def add_param_group(self, group) -> None:
        super().add_param_group(group)
        for p in self.param_groups[-1]["params"]:
            if p.dim() < 2:
                self.param_groups.pop()
                raise ValueError(f"Muon: parameters have two axes or more, got one of shape {tuple(p.shape)}")

    @torch.no_grad()
    def step(self, closure=None) -> Optional[torch.Tensor]:
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        # what is refused is refused before anything has changed
        for group, sets in [(group, self._sets(group)) for group in self.param_groups]:
            for (shape, dtype, _), params in sets.items():
                wide = dtype == torch.float32
                grads = [p.grad for p in params] if wide else list(torch.stack([p.grad for p in params]).float().unbind(0))
                held = [self._momentum(p) for p in params]
                torch._foreach_mul_(held, group["momentum"])
                torch._foreach_add_(held, grads)
                update = torch._foreach_add(grads, held, alpha=group["momentum"]) if group["nesterov"] else held
                turned = orthogonalize(torch.stack(update), group["steps"], group["coefficients"], group["eps"])
                keep, by = 1.0 - group["lr"] * group["weight_decay"], -group["lr"] * max(1.0, shape[-2] / max(shape[-1], 1)) ** 0.5
                if wide:
                    if group["weight_decay"]:
                        torch._foreach_mul_(params, keep)
                    torch._foreach_add_(params, list(turned.unbind(0)), alpha=by)
                else:
                    new = torch.stack(params).float().mul_(keep).add_(turned, alpha=by)
                    torch._foreach_copy_(params, list(new.unbind(0)))
        return loss

    @staticmethod
    def _sets(group) -> dict:
        """The parameters of a group that have a gradient, by shape, type and device."""
        sets = {}
        for p in group["params"]:
            if p.grad is not None:
                if p.grad.is_sparse:
                    raise RuntimeError("Muon: sparse gradients are not supported")
                if p.dtype not in (torch.float32, torch.bfloat16, torch.float16):
                    raise RuntimeError(f"Muon: parameters are float32, bfloat16 or float16, got {p.dtype}")
                sets.setdefault((p.shape, p.dtype, p.device), []).append(p)
        for (shape, _, device), params in sets.items():
            if shape.numel() and len(params) * math.prod(shape[:-2]) > 65535:
                raise RuntimeError(f"Muon: at most 65535 matrices of one shape, got {len(params)} parameters of {tuple(shape)}")
            orthogonalize(torch.empty((0, *shape[-2:]), device=device), group["steps"], group["coefficients"], group["eps"])      # the checks alone
        return sets

    def _momentum(self, p: torch.Tensor) -> torch.Tensor:
        state = self.state[p]
        if "momentum_buffer" not in state:
            state["momentum_buffer"] = torch.zeros_like(p, dtype=torch.float32)
        elif state["momentum_buffer"].dtype != torch.float32:
            state["momentum_buffer"] = state["momentum_buffer"].float()
        return state["momentum_buffer"]

    def load_state_dict(self, state_dict) -> None:
        """As that of any optimiser, which gives the state the parameters' types; the momentum of 16-bit ones is taken over in fp32."""
        super().load_state_dict(state_dict)
        ids = [i for group in state_dict["param_groups"] for i in group["params"]]
        for i, p in zip(ids, (p for group in self.param_groups for p in group["params"])):
            held = state_dict["state"].get(i, {}).get("momentum_buffer")
            if held is not None and p.dtype != torch.float32:
                self.state[p]["momentum_buffer"] = held.to(device=p.device, dtype=torch.float32, copy=True)
