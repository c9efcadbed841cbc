"""The root-mean-square norm in front of a layer, as a module."""

import torch

from fast_llm_amd.functional.normalization import rms_norm


class RMSNorm(torch.nn.Module):
    """`rms_norm` with its weight. Also fits `DroplessMoEMLP`'s `router_normalization`."""

    def __init__(
        self,
        hidden_size: int,
        eps: float = 1e-5,
        *,
        dtype: torch.dtype = torch.bfloat16,
        device: torch.device | str = "cuda",
    ):
        super().__init__()
        self.eps = eps
        self.weight = torch.nn.Parameter(torch.ones(hidden_size, dtype=dtype, device=device))

    def forward(
        self, input_: torch.Tensor, residual: torch.Tensor | None = None
    ) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
        """The normalised input; with a residual, which is added first, also the sum that goes on (`normalized`, `stream`)."""
        return rms_norm(input_, self.weight, residual, self.eps)
