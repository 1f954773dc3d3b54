"""y = x Wᵀ for a weight kept [out, in] as the checkpoint stores it (no transposes:
AntoineBut/TileInfer.jl src/hub/loader.jl:1-6), 32-bit accumulation and one rounding
(src/ops/reference.jl:23-26). The kernel is chosen by element type, token count and sizes;
the 32-bit path always takes the CUDA-core product."""
from __future__ import annotations

import torch

from ..kernels import ops


class Linear:
    def __init__(self, weight: torch.Tensor, rt, name: str = "linear"):
        self.rt = rt
        self.weight = weight                 # [out, in], compute dtype, on the device
        self.out_features, self.in_features = weight.shape
        self.name = name
        # Where split-k partial sums go; two products whose partial sums are alive at the same time name different buffers.
        self.partials_name = "linear.partials"

    def forward(self, x: torch.Tensor, out: torch.Tensor, epilogue: int = ops.EPI_NONE, act=(0.0, 0.0, 0.0, 0.0),
                allow_partials: bool = False):
        """Writes y to ``out`` and returns it. With ``allow_partials`` the result may instead come back
        as 32-bit partial sums ``[s, n, out]`` (a product split over k), for a consumer that adds them:
        the norm's ``add_forward``."""
        if self.rt.fast:
            from ..kernels import fast
            done = fast.linear(self, x, out, epilogue, act, allow_partials)
            if done is not None:
                return done
        ops.gemm_plain(out, x, self.weight, epilogue, act)
        return out

    def forward_f32(self, x: torch.Tensor, out: torch.Tensor):
        """Writes the 32-bit sums to ``out`` [n, out] float32, not rounded to the element type where a fast kernel takes the sizes."""
        if self.rt.fast:
            from ..kernels import fast
            done = fast.linear_f32(self, x, out)
            if done is not None:
                return done
        ops.gemm_plain(out, x, self.weight, ops.EPI_F32_OUT)
        return out


class Linear4(Linear):
    """The same product with a matrix of 4 bits a weight, made from another's: codes with a scale (and, asked for, a zero) per group of ``group``
    inputs, or of the largest smaller group that divides them. Nothing of the other is kept; there is no ``weight``."""

    def __init__(self, other: Linear, group: int = 128, zeros: bool = False):
        fit = next((g for g in sorted(ops.LINEAR4_GROUPS, reverse=True) if g <= group and other.in_features % g == 0), None)
        if fit is None:
            raise ValueError(f"{other.name}: {other.in_features} inputs do not divide into groups of {', '.join(map(str, ops.LINEAR4_GROUPS))} up to {group}")
        self.rt, self.name, self.partials_name = other.rt, other.name, other.partials_name
        self.out_features, self.in_features, w = other.out_features, other.in_features, other.weight
        groups = self.in_features // fit
        self.codes = torch.empty(self.out_features, self.in_features // 8, dtype=torch.int32, device=w.device)
        self.scales = torch.empty(groups, self.out_features, dtype=w.dtype, device=w.device)
        self.zeros = torch.empty(groups, self.out_features, dtype=torch.uint8, device=w.device) if zeros else None
        ops.quantize4(self.codes, self.scales, w, self.zeros)

    def forward(self, x: torch.Tensor, out: torch.Tensor, epilogue: int = ops.EPI_NONE, act=(0.0, 0.0, 0.0, 0.0), allow_partials: bool = False):
        ops.linear4(out, x, self.codes, self.scales, self.zeros, epilogue, act, self._workspace(x.shape[0]))
        return out

    def forward_f32(self, x: torch.Tensor, out: torch.Tensor):
        ops.linear4(out, x, self.codes, self.scales, self.zeros, ops.EPI_F32_OUT, workspace=self._workspace(x.shape[0]))
        return out

    def _workspace(self, n: int):
        need = ops.linear4_workspace(n, self.out_features, self.in_features) if self.rt.dtype == torch.bfloat16 else 0
        return self.rt.buffer("linear4.parts", (need,), torch.uint8) if need else None
