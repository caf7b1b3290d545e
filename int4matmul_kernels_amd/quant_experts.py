"""Caller-side modules of a mixture of experts whose weights live in the packed formats.

``ExpertRouter`` turns a router's logits into each token's experts and their weights
(``int4matmul.route_experts``); ``QuantExperts`` holds the experts' packed matrices, as
``QuantLinear`` holds one layer's, and applies the gated feed-forward of the experts that each
token was given (``int4matmul.experts_forward``).  No counterpart in the reference, whose every
product takes one matrix.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

import int4matmul_kernels_amd as pkg
from int4matmul_kernels_amd.quant_linear import QuantLinear


class ExpertRouter(torch.nn.Module):
    """logits ``[..., n_experts]`` (fp16 or fp32) -> ``(weights, ids)``, fp32 and int32 ``[..., top_k]``, best first.

    Scores are the softmax or the sigmoid of the logits; an expert whose logit is -inf or NaN is out.  The ``top_k``
    best are taken, by score or with ``bias=True`` by score plus ``self.bias`` (fp32, not part of the weights), ties to
    the lowest index.  With ``n_groups`` groups of neighbouring experts only those of the ``topk_groups`` best groups are
    eligible, by their best (``group_score="max"``) or the sum of their two best (``"top2"``).  Weights are the scores,
    divided by their sum if ``renormalize``, times ``scale``.  Where fewer experts are left than ``top_k``, the last ids
    are -1 and their weights 0.
    """

    def __init__(self, n_experts: int, top_k: int, scoring: str = "softmax", bias: bool = False, n_groups: int = 1,
                 topk_groups: int = 1, group_score: str = "max", renormalize: bool = True, scale: float = 1.0, device="cuda"):
        super().__init__()
        if not 1 <= n_experts <= 1024:
            raise ValueError("n_experts must be 1 ... 1024")
        if not 1 <= n_groups <= 64 or n_experts % n_groups or not 1 <= topk_groups <= n_groups:
            raise ValueError("n_groups (up to 64) must divide n_experts, and topk_groups be 1 ... n_groups")
        if not 1 <= top_k <= min(64, n_experts // n_groups * topk_groups):
            raise ValueError("top_k must be 1 ... 64 and no more than the experts of topk_groups groups")
        if scoring not in ("softmax", "sigmoid"):
            raise ValueError('scoring must be "softmax" or "sigmoid"')
        if group_score not in ("max", "top2"):
            raise ValueError('group_score must be "max" or "top2"')
        self.n_experts, self.top_k, self.scoring, self.n_groups = n_experts, top_k, scoring, n_groups
        self.topk_groups, self.group_score, self.renormalize, self.scale = topk_groups, group_score, renormalize, scale
        self.register_buffer("bias", torch.zeros((n_experts,), dtype=torch.float32, device=device) if bias else None)

    def _apply(self, fn, recurse=True):
        # half() and the like leave the bias alone: it is fp32 in every model
        bias = self.bias
        super()._apply(fn, recurse)
        if bias is not None and self.bias.dtype != torch.float32:
            self.bias = bias.to(self.bias.device)
        return self

    def forward(self, logits: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        if logits.shape[-1] != self.n_experts:
            raise ValueError(f"logits must be [..., {self.n_experts}] but are {tuple(logits.shape)}")
        return pkg.load_extension().route_experts(logits, self.top_k, self.scoring, self.bias, self.n_groups, self.topk_groups,
                                                  self.group_score, self.renormalize, self.scale)

    def extra_repr(self) -> str:
        return (f"n_experts={self.n_experts}, top_k={self.top_k}, scoring={self.scoring}, n_groups={self.n_groups}, "
                f"topk_groups={self.topk_groups}, group_score={self.group_score}, renormalize={self.renormalize}, scale={self.scale}")


class QuantExperts(torch.nn.Module):
    """``y[t] = sum_j weights[t, j] * (silu(x[t] @ gate_e) * (x[t] @ up_e)) @ down_e``, ``e = ids[t, j]``; an id outside
    ``0 ... n_experts - 1`` adds nothing.

    ``up_*`` hold ``[n_experts, ..., 2 * width]`` packed matrices of ``features`` inputs, gate columns first, ``down_*``
    ``[n_experts, ..., features]`` ones of ``width`` inputs; the formats are ``QuantLinear``'s.
    """

    def __init__(self, bits: int, n_experts: int, features: int, width: int, group_size: int = 128, sparse: bool = False, device="cuda"):
        super().__init__()
        if bits not in (4, 3, 2):
            raise ValueError("bits must be 4, 3 or 2")
        if sparse and bits != 4:
            raise ValueError("16:32 sparsity is supported for int4 only")
        if n_experts < 1:
            raise ValueError("n_experts must be positive")
        if features % 64 or width % 64 or features < 64 or width < 64:
            raise ValueError("features and width must be positive multiples of 64")
        if group_size == 0 or (group_size > 0 and group_size % 64):
            raise ValueError("group_size must be negative or a positive multiple of 64")
        self.bits, self.n_experts, self.features, self.width = bits, n_experts, features, width
        self.group_size, self.sparse = group_size, sparse
        for name, k, s in (("up", features, 2 * width), ("down", width, features)):
            rows = k // 16 if sparse else k * bits // 32
            groups = 1 if group_size < 0 else (k + group_size - 1) // group_size
            self.register_buffer(f"{name}_matrix", torch.zeros((n_experts, rows, s), dtype=torch.int32, device=device))
            self.register_buffer(f"{name}_scales", torch.ones((n_experts, groups, s), dtype=torch.float16, device=device))
            self.register_buffer(f"{name}_zeros", torch.zeros((n_experts, groups, s), dtype=torch.float16, device=device))
            self.register_buffer(f"{name}_mask", torch.zeros((n_experts, k // 32, s), dtype=torch.int32, device=device) if sparse else None)

    @torch.no_grad()
    def set_expert(self, expert: int, up: QuantLinear, down: QuantLinear) -> None:
        """fills one expert from two packed layers: ``up`` [features, 2 * width] (gate columns first), ``down`` [width, features]"""
        if not 0 <= expert < self.n_experts:
            raise IndexError(f"expert {expert} of {self.n_experts}")
        for name, layer, k, s in (("up", up, self.features, 2 * self.width), ("down", down, self.width, self.features)):
            if (layer.bits, layer.in_features, layer.out_features, layer.group_size, layer.sparse) != (self.bits, k, s, self.group_size, self.sparse):
                raise ValueError(f"{name} does not match: {layer.extra_repr()}")
            if layer.bias is not None:
                raise ValueError("experts have no bias")
            for part in ("matrix", "scales", "zeros") + (("mask",) if self.sparse else ()):
                mine = getattr(self, f"{name}_{part}")[expert]
                mine.copy_(getattr(layer, "sparse_mask" if part == "mask" else part).reshape(mine.shape))

    @classmethod
    def from_float(cls, up: torch.Tensor, down: torch.Tensor, bits: int = 4, group_size: int = 128, up_keep: Optional[torch.Tensor] = None,
                   down_keep: Optional[torch.Tensor] = None):
        """``QuantLinear.from_float`` of every expert's ``up`` ``[n_experts, features, 2 * width]`` and ``down``
        ``[n_experts, width, features]``; ``*_keep`` (bool, the same shapes) selects the 16:32 format"""
        if (up_keep is None) != (down_keep is None):
            raise ValueError("16:32 experts need both masks")
        n, features, columns = up.shape
        m = cls(bits, n, features, columns // 2, group_size, up_keep is not None, device=up.device)
        for e in range(n):
            m.set_expert(e, QuantLinear.from_float(up[e], bits, group_size, None if up_keep is None else up_keep[e]),
                         QuantLinear.from_float(down[e], bits, group_size, None if down_keep is None else down_keep[e]))
        return m

    def forward(self, x: torch.Tensor, weights: torch.Tensor, ids: torch.Tensor) -> torch.Tensor:
        """``x`` ``[..., features]`` with a router's ``weights`` and ``ids`` ``[..., top_k]``"""
        return pkg.load_extension().experts_forward(self.bits, x, weights, ids, self.up_matrix, self.up_scales, self.up_zeros,
                                                    self.down_matrix, self.down_scales, self.down_zeros, self.group_size, self.up_mask,
                                                    self.down_mask)

    def extra_repr(self) -> str:
        return (f"bits={self.bits}, n_experts={self.n_experts}, features={self.features}, width={self.width}, "
                f"group_size={self.group_size}, sparse={self.sparse}")
