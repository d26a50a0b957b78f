"""Muon: momentum whose matrix updates are orthogonalised before they are
applied (``orthogonalize``, Newton-Schulz on the tensor cores).

For weight matrices and stacks of them ([..., rows, cols], such as the
promotion parameters [L - 1, H, K, V]); embeddings, norms and other vectors
belong to an elementwise optimiser beside it (``split_parameters``).
"""

from __future__ import annotations

import torch

from .orthogonal import orthogonalize

__all__ = ["Muon", "split_parameters"]


def split_parameters(model):
    """(matrices for Muon, everything else) of a model: the weights of linear
    layers and stacked projections, but neither embeddings nor the LM head
    nor depthwise convolutions."""
    matrices, rest = [], []
    for name, p in model.named_parameters():
        matrix = p.dim() >= 2 and min(p.shape[-2:]) > 1 and not any(
            part in name for part in ("embeddings", "lm_head", "conv1d"))
        (matrices if matrix else rest).append(p)
    return matrices, rest


class Muon(torch.optim.Optimizer):
    """``buf = momentum * buf + grad``; the update is the orthogonalised
    ``grad + momentum * buf`` (``nesterov``) or ``buf``, times
    ``sqrt(max(1, rows / cols))``. Momenta are float32. Updates of one shape
    are orthogonalised in one call."""

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, steps=5, weight_decay=0.0):
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, steps=steps,
                                      weight_decay=weight_decay))
        for group in self.param_groups:
            for p in group["params"]:
                if p.dim() < 2:
                    raise ValueError(f"Muon takes matrices [..., rows, cols], got {tuple(p.shape)}")

    def load_state_dict(self, state_dict):
        """As torch's, which casts a state to its parameter's type; momenta stay
        float32."""
        super().load_state_dict(state_dict)
        for saved, group in zip(state_dict["param_groups"], self.param_groups):
            for i, p in zip(saved["params"], group["params"]):
                if "momentum" in state_dict["state"].get(i, ()):
                    self.state[p]["momentum"] = state_dict["state"][i]["momentum"].to(
                        device=p.device, dtype=torch.float32, copy=True,
                        memory_format=torch.contiguous_format)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            by_shape = {}
            for p in group["params"]:
                if p.grad is not None:
                    by_shape.setdefault((p.shape, p.device, p.dtype), []).append(p)
            for ps in by_shape.values():
                updates = []
                for p in ps:
                    state = self.state[p]
                    if "momentum" not in state:
                        state["momentum"] = torch.zeros_like(p, dtype=torch.float32,
                                                             memory_format=torch.contiguous_format)
                    grad, buf = p.grad.float(), state["momentum"]
                    buf.mul_(group["momentum"]).add_(grad)
                    updates.append(grad.add(buf, alpha=group["momentum"]) if group["nesterov"] else buf)
                dtype = ps[0].dtype if ps[0].dtype != torch.float32 else torch.bfloat16
                ortho = orthogonalize(torch.stack(updates), steps=group["steps"], dtype=dtype)
                rows, cols = ps[0].shape[-2:]
                scale = max(1.0, rows / cols) ** 0.5
                for p, u in zip(ps, ortho):
                    if group["weight_decay"]:
                        p.mul_(1.0 - group["lr"] * group["weight_decay"])
                    p.add_(u, alpha=-group["lr"] * scale)
        return loss
