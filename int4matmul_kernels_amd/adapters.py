"""Low-rank adapters of many requests beside a projection that they share.

``LowRankAdapters`` holds the factors of ``n_adapters`` adapters of one layer; ``QuantLinear`` adds them onto its
output: ``layer(x, adapters, ids)`` is ``x @ W_q + scales[a] * (x @ down[a].T) @ up[a] (+ bias)`` with each row's own
``a``.  No counterpart in the reference.
"""
from __future__ import annotations

from typing import Optional

import torch

import int4matmul_kernels_amd as pkg


class LowRankAdapters(torch.nn.Module):
    """``down`` fp16 ``[n_adapters, rank, in_features]``, ``up`` fp16 ``[n_adapters, rank, out_features]``, ``scales`` fp32
    ``[n_adapters]``; an adapter of a lower rank has zeros in its last ranks."""

    def __init__(self, n_adapters: int, rank: int, in_features: int, out_features: int, device="cuda"):
        super().__init__()
        if n_adapters < 1:
            raise ValueError("n_adapters must be positive")
        if not 1 <= rank <= 512:
            raise ValueError("rank must be 1 ... 512")
        if in_features % 64 or out_features % 64 or in_features < 64 or out_features < 64:
            raise ValueError("in_features and out_features must be positive multiples of 64")
        self.n_adapters, self.rank, self.in_features, self.out_features = n_adapters, rank, in_features, out_features
        self.register_buffer("down", torch.zeros((n_adapters, rank, in_features), dtype=torch.float16, device=device))
        self.register_buffer("up", torch.zeros((n_adapters, rank, out_features), dtype=torch.float16, device=device))
        self.register_buffer("scales", torch.zeros((n_adapters,), dtype=torch.float32, device=device))

    def _apply(self, fn, recurse=True):
        # half() and the like turn the factors alone: the scales are fp32 in every model
        scales = self.scales
        super()._apply(fn, recurse)
        if self.scales.dtype != torch.float32:
            self.scales = scales.to(self.scales.device)
        return self

    @torch.no_grad()
    def set_adapter(self, index: int, down: torch.Tensor, up: torch.Tensor, scale: float = 1.0) -> None:
        """fills one adapter from its factors ``down`` ``[rank, in_features]`` and ``up`` ``[out_features, rank]``, of this rank or a lower one"""
        if not 0 <= index < self.n_adapters:
            raise IndexError(f"adapter {index} of {self.n_adapters}")
        rank = down.shape[0]
        if not 1 <= rank <= self.rank or tuple(down.shape) != (rank, self.in_features) or tuple(up.shape) != (self.out_features, rank):
            raise ValueError(f"factors must be [r, {self.in_features}] and [{self.out_features}, r] with r up to {self.rank} but are "
                             f"{tuple(down.shape)} and {tuple(up.shape)}")
        self.down[index, :rank].copy_(down)
        self.up[index, :rank].copy_(up.t())
        self.down[index, rank:].zero_()
        self.up[index, rank:].zero_()
        self.scales[index] = scale

    def forward(self, base: torch.Tensor, x: torch.Tensor, ids: torch.Tensor, outs: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``base`` ``[..., out_features]`` plus each row's adapter applied to ``x`` ``[..., in_features]``.  ``ids`` (int32) are
        ``x``'s leading sizes, one or more of them: one id per request or one per row; an id outside ``0 ... n_adapters - 1``
        is no adapter.  ``outs`` may be ``base``."""
        return pkg.load_extension().low_rank_add(base, x, self.down, self.up, self.scales, ids, outs)

    def extra_repr(self) -> str:
        return f"n_adapters={self.n_adapters}, rank={self.rank}, in_features={self.in_features}, out_features={self.out_features}"
