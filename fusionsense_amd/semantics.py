"""Class scores on the Gaussians: the head that turns a rendered feature plane into scores.

The reference's active-touch module names an object's parts, segments views of it with a 2-D model and fuses the labels with
the high-gradient points (scripts/VLM.py:55-385); its Gaussians carry no labels.  Here every Gaussian carries a feature row
``gauss_params["semantics"]`` [N,D]; :func:`fusionsense_amd.fusion.render_fusionsense` composites it to a plane like a colour
and hands that plane to a :class:`SemanticHead`; :func:`fusionsense_amd.losses.topk_distill_loss` trains both against what was
kept of a 2-D teacher's scores.  The same head on the feature rows themselves labels the points to touch.

The rows and the head are the caller's to optimize: ``SplatTrainer`` takes the reference's parameters only, so train them on
Gaussians that are no longer split or culled (each of those leaves N, and with it the rows, behind)."""
from __future__ import annotations

import math
from typing import Optional

import torch
from torch import Tensor

from . import ops


class SemanticHead(torch.nn.Module):
    """``in_dim`` features -> ``n_classes`` scores: one layer to ``hidden`` channels, ``blocks`` residual layers of that width,
    a class layer; every layer is one ``ops.linear_act`` launch.  ``hidden = 0``: the class layer alone.  The parameters'
    ``dtype`` is the type the head computes in; features of another type are cast to it."""

    def __init__(self, in_dim: int, n_classes: int, hidden: int = 64, blocks: int = 1, act: str = "gelu",
                 dtype: torch.dtype = torch.float32, device=None, generator: Optional[torch.Generator] = None):
        super().__init__()
        if dtype not in ops.DTYPES:
            raise ValueError(f"dtype must be float32, bfloat16 or float16, got {dtype}")
        if act not in ops.ACTIVATIONS:
            raise ValueError(f"act must be one of {tuple(ops.ACTIVATIONS)}, got {act!r}")
        if hidden < 0 or blocks < 0 or in_dim < 1 or n_classes < 1 or (hidden == 0 and blocks > 0):
            raise ValueError(f"no head of {in_dim} -> {hidden} x {blocks} -> {n_classes}")
        self.act = act
        widths = [in_dim] + ([hidden] * (1 + blocks) if hidden else []) + [n_classes]
        self.weights, self.biases = torch.nn.ParameterList(), torch.nn.ParameterList()
        for k, n in zip(widths[:-1], widths[1:]):
            bound = 1.0 / math.sqrt(k)  # (drawn on the CPU: the same generator gives the same head on every device)
            w = (torch.rand(n, k, generator=generator) * 2 - 1) * bound
            b = (torch.rand(n, generator=generator) * 2 - 1) * bound
            self.weights.append(torch.nn.Parameter(w.to(device=device, dtype=dtype)))
            self.biases.append(torch.nn.Parameter(b.to(device=device, dtype=dtype)))

    def forward(self, features: Tensor) -> Tensor:
        h = features.to(self.weights[0].dtype)
        last = len(self.weights) - 1
        for i, (w, b) in enumerate(zip(self.weights, self.biases)):
            if i == last:
                return ops.linear_act(h, w, b)
            h = ops.linear_act(h, w, b, self.act, residual=h if i > 0 else None)
