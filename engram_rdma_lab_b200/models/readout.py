"""The read-out of one layer's looked-up rows: layer norm, then a projection to the model's features.

``EngramReadout`` takes what ``EngramBuffer.fetch`` returns for a layer, ``data [tokens, hidden * entries]`` in bf16
or ``(data, scales)`` in e4m3, and gives ``[tokens, features]``.  In training one 8-bit checkpoint of the normalised
rows serves both backward passes (:func:`engram_rdma_lab_b200.ops.norm_linear`), and nothing else of the lookup's
size is kept, so the buffer is free for the next fetch as soon as the forward pass has run.
"""

from __future__ import annotations

import torch

from ..ops import norm_linear


class EngramReadout(torch.nn.Module):
    """``layer_norm(rows) @ weight^T + bias`` for rows of ``entries`` looked-up rows of ``hidden`` columns each.

    ``block`` is the columns per scale of e4m3 tables.  Parameters have ``dtype``, and so has the result (autocast's
    type under autocast): rows of that type, e4m3 codes with their scales or, with fp32 parameters, bf16 and fp16 rows,
    which are widened first (exactly, and not kept).
    """

    def __init__(self, hidden: int, entries: int, features: int, *, bias: bool = False, eps: float = 1e-5,
                 block: int = 128, dtype: torch.dtype = torch.bfloat16, device=None):
        super().__init__()
        if min(hidden, entries, features) < 1:
            raise ValueError("hidden, entries and features must be positive")
        self.hidden, self.entries, self.features, self.eps, self.block = hidden, entries, features, eps, block
        width = hidden * entries
        self.norm_weight = torch.nn.Parameter(torch.ones(width, dtype=dtype, device=device))
        self.norm_bias = torch.nn.Parameter(torch.zeros(width, dtype=dtype, device=device))
        self.weight = torch.nn.Parameter(torch.empty(features, width, dtype=dtype, device=device))
        self.bias = torch.nn.Parameter(torch.zeros(features, dtype=dtype, device=device)) if bias else None
        torch.nn.init.normal_(self.weight, std=width ** -0.5)

    def forward(self, data: torch.Tensor, scales: torch.Tensor | None = None) -> torch.Tensor:
        lookup = {} if scales is None else dict(scales=scales, hidden=self.hidden, block=self.block,
                                                dtype=self.weight.dtype)
        if scales is None and self.weight.dtype == torch.float32 and data.dtype in (torch.bfloat16, torch.float16):
            data = data.float()
        return norm_linear(data, self.norm_weight, self.norm_bias, self.weight, self.bias, self.eps, **lookup)
