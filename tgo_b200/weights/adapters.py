"""Low-rank adapters of a model: reading them, checking them against the model's products, and laying
all of them out together.

An adapter changes a product's matrix W [out, in] to W + scale * B A, A [rank, in], B [out, rank]. On
disk it is a folder with `adapter_config.json` (r, lora_alpha, use_rslora; scale = alpha / r, or alpha /
sqrt(r)) and `adapter_model.safetensors`, tensors `<matrix>.lora_A.weight` and `<matrix>.lora_B.weight`,
`<matrix>` being the checkpoint's name of W without `.weight`, with or without the prefix
`base_model.model.`. In memory it is {matrix name: (A, B)} and a scale.

The adapters of a site (parts/base.py: AdapterSite) become one bank: A [adapters, slices, rank, in] and
B [adapters, columns, rank], in the engine's type, the rank the largest among them in whole fours and the rest
zeros, B's rows in the order of the product's columns.
"""
from __future__ import annotations

import json
import math
import os
from dataclasses import dataclass
from typing import Dict, List, Tuple

import torch

from ..parts.base import AdapterBank, AdapterSite
from .safetensors import SafetensorsFile

PREFIX = "base_model.model."
MAX_ADAPTERS = 3071               # one bank's; the kernels' plan of a step's rows holds as many


class AdapterError(ValueError):
    pass


@dataclass
class Adapter:
    """`matrices`: checkpoint name of a matrix (with `.weight`) -> (A [rank, in], B [out, rank])."""
    matrices: Dict[str, Tuple[torch.Tensor, torch.Tensor]]
    scale: float = 1.0


def read_adapter(folder: str) -> Adapter:
    """The adapter of a folder; whatever it holds that this engine would not apply is refused."""
    with open(os.path.join(folder, "adapter_config.json")) as f:
        config = json.load(f)
    rank, alpha = config.get("r"), config.get("lora_alpha")
    if not isinstance(rank, int) or isinstance(rank, bool) or rank <= 0:
        raise AdapterError(f"adapter {folder}: adapter_config.json: r is {rank!r}; a positive whole number is needed")
    if not isinstance(alpha, (int, float)) or isinstance(alpha, bool) or not math.isfinite(alpha):
        raise AdapterError(f"adapter {folder}: adapter_config.json: lora_alpha is {alpha!r}; a number is needed")
    for key, plain in (("use_dora", (None, False)), ("bias", (None, "none")), ("modules_to_save", (None, [])),
                       ("rank_pattern", (None, {})), ("alpha_pattern", (None, {})), ("fan_in_fan_out", (None, False))):
        if config.get(key) not in plain:
            raise AdapterError(f"adapter {folder}: adapter_config.json: {key} = {config[key]!r} is not supported")
    # how the halves were begun matters only where the model's own matrices were changed for it
    if config.get("init_lora_weights") not in (None, True, False, "gaussian", "eva", "orthogonal"):
        raise AdapterError(f"adapter {folder}: adapter_config.json: init_lora_weights = {config['init_lora_weights']!r}: the halves "
                           "may belong to matrices that were changed when they were begun")
    scale = alpha / math.sqrt(rank) if config.get("use_rslora") else alpha / rank
    file = SafetensorsFile(os.path.join(folder, "adapter_model.safetensors"))
    halves: Dict[str, Dict[str, torch.Tensor]] = {}
    strange = []
    try:
        for name in file.entries:
            plain = name[len(PREFIX):] if name.startswith(PREFIX) else name
            for half in ("A", "B"):
                end = f".lora_{half}.weight"
                if plain.endswith(end):
                    halves.setdefault(plain[:-len(end)] + ".weight", {})[half] = file.tensor(name).clone()
                    break
            else:
                strange.append(name)
    finally:
        file.close()
    if strange:
        raise AdapterError(f"adapter {folder}: tensors that are no half of a low-rank matrix: {sorted(strange)[:5]}")
    lone = sorted(m for m, h in halves.items() if len(h) != 2)
    if lone:
        raise AdapterError(f"adapter {folder}: only one of lora_A and lora_B is there for {lone[:5]}")
    return Adapter({m: (h["A"], h["B"]) for m, h in halves.items()}, scale)


def _check(name: str, adapter: Adapter, sites: Dict[str, Tuple[AdapterSite, int]], dtype) -> None:
    """One error that lists everything an adapter and the model disagree on. Its numbers have to be finite as the
    engine holds them: the matrices in `dtype`, the scale in float32."""
    wrong = []
    if not adapter.matrices:
        wrong.append("it holds no matrices")
    if not bool(torch.isfinite(torch.tensor(adapter.scale, dtype=torch.float64).float())):
        wrong.append(f"its scale is {adapter.scale}")
    for matrix, (a, b) in sorted(adapter.matrices.items()):
        if matrix not in sites:
            wrong.append(f"{matrix} is no product of this model that an adapter can add to")
            continue
        site, i = sites[matrix]
        if a.dim() != 2 or b.dim() != 2 or a.shape[0] != b.shape[1] or a.shape[0] == 0 or \
                a.shape[1] != site.inputs or b.shape[0] != site.widths[i]:
            wrong.append(f"{matrix}: A {list(a.shape)} and B {list(b.shape)} for a matrix of "
                         f"[{site.widths[i]}, {site.inputs}]")
        elif not (a.is_floating_point() and b.is_floating_point()):
            wrong.append(f"{matrix}: A and B hold whole numbers")
        elif not (bool(torch.isfinite(a.to(dtype)).all()) and bool(torch.isfinite(b.to(dtype)).all())):
            wrong.append(f"{matrix}: A or B holds a number that is not finite in {dtype}")
    if wrong:
        raise AdapterError(f"adapter {name!r}: " + "; ".join(wrong[:8]) + ("; ..." if len(wrong) > 8 else ""))


def _bank(site: AdapterSite, adapters: List[Adapter], dtype, device) -> AdapterBank:
    n, S, N = len(adapters), len(site.widths), sum(site.widths)
    rank = max(a.shape[0] for ad in adapters for m in site.names if m in ad.matrices for a in [ad.matrices[m][0]])
    rank = (rank + 3) // 4 * 4
    a = torch.zeros((n, S, rank, site.inputs), dtype=dtype, device=device)
    b = torch.zeros((n, N, rank), dtype=dtype, device=device)
    first = 0
    for s, (matrix, width) in enumerate(zip(site.names, site.widths)):
        if site.interleaved:
            columns = torch.arange(width, device=device)
            columns = columns // 8 * 16 + s * 8 + columns % 8
        else:
            columns = torch.arange(first, first + width, device=device)
        for i, ad in enumerate(adapters):
            if matrix in ad.matrices:
                half_a, half_b = ad.matrices[matrix]
                r = half_a.shape[0]
                a[i, s, :r] = half_a.to(device=device, dtype=dtype)
                b[i, columns, :r] = half_b.to(device=device, dtype=dtype)
        first += width
    scale = torch.tensor([ad.scale for ad in adapters], dtype=torch.float32, device=device)
    return AdapterBank(a, b, scale, tuple(site.widths), site.interleaved)


def bind_adapters(model, adapters: Dict[str, Adapter]) -> List[str]:
    """Check every adapter against the model's products, lay them out and hand each part its banks. Returns
    the adapters' names in the order of their numbers."""
    if len(adapters) > MAX_ADAPTERS:
        raise AdapterError(f"{len(adapters)} adapters; at most {MAX_ADAPTERS} are held together")
    parts = [p for block in model.blocks for p in (block.parts() if hasattr(block, "parts") else [block])]
    parts = [(p, p.adapter_sites()) for p in parts if hasattr(p, "adapter_sites") and hasattr(p, "bind_adapters")]
    sites = {m: (s, i) for _, own in parts for s in own for i, m in enumerate(s.names)}
    for name, adapter in adapters.items():
        _check(name, adapter, sites, model.dtype)
    every = list(adapters.values())
    for part, own in parts:
        part.bind_adapters({s.key: _bank(s, every, model.dtype, model.device) for s in own
                            if any(m in ad.matrices for ad in every for m in s.names)})
    return list(adapters)
