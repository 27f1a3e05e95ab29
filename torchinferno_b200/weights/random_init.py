"""Random weights: every matrix N(0, std), norm vectors 1 (or 1 + N(0, std) where a part asks for it; small square
matrices of coefficients the unit matrix + N(0, std)), from a seed.

Each tensor has a generator of its own, keyed by (seed, tensor name), so a
tensor's values do not depend on which other tensors exist or on their order.
The reference has no such mode; its tests build an eager model under
``torch.manual_seed`` and write it out to load it back
(tests/test_model_variants.py:319-354 in the reference project).

With ``quantization_config`` in config.json (config/quantization.py) the matrices it covers are quantised to 8-bit blocks; where it names
a form that is not read, random weights are of the model's own type, as without it.
"""
from __future__ import annotations

import hashlib
import json
from pathlib import Path
from typing import Any, Mapping

import torch

from torchinferno_b200.config.model_config import ConfigError
from torchinferno_b200.config.quantization import SCALE_SUFFIX, BlockQuantization
from torchinferno_b200.config.registry import resolve_architecture
from torchinferno_b200.kernels.block_scaled import quantize_matrix
from torchinferno_b200.weights.loader import SINGLE_FILE, place, place_blocks


def _tensor_seed(seed: int, name: str) -> int:
    digest = hashlib.sha256(f"{seed}:{name}".encode()).digest()
    return int.from_bytes(digest[:8], "little") & 0x7FFF_FFFF_FFFF_FFFF


def random_tensor(spec, seed: int, *, device: torch.device | str = "cpu",
                  dtype: torch.dtype = torch.float32) -> torch.Tensor:
    if spec.init == "ones":
        return torch.ones(spec.shape, dtype=dtype, device=device)
    if spec.init == "zeros":
        return torch.zeros(spec.shape, dtype=dtype, device=device)
    if spec.init not in ("normal", "about_one", "about_identity"):
        raise ValueError(f"unknown init {spec.init!r} for {spec.name}")
    generator = torch.Generator(device=device)
    generator.manual_seed(_tensor_seed(seed, spec.name))
    out = torch.empty(spec.shape, dtype=torch.float32, device=device)
    out.normal_(0.0, spec.std, generator=generator)
    if spec.init == "about_one":
        out += 1.0
    if spec.init == "about_identity":          # (a square matrix: the unit matrix plus noise)
        out += torch.eye(spec.shape[0], spec.shape[1], device=device)
    return out.to(dtype)


def build_model(config: Mapping[str, Any], *, dtype: torch.dtype, device: torch.device | str):
    """The model that ``config`` (a config.json as a dict) names, without weights."""
    from torchinferno_b200.models.model import CausalLM
    entry = resolve_architecture(config)
    typed = entry.config_class.from_dict(config)
    return CausalLM(entry.build(typed), dtype=dtype, device=device)


def _quantization(config: Mapping[str, Any]) -> BlockQuantization | None:
    """What config.json has stored in 8-bit blocks.  (A form of 8-bit weights that is not read concerns files, and their loader: a random model has none.)"""
    try:
        return BlockQuantization.from_config(config)
    except ConfigError:
        return None


def _in_blocks(quantization: BlockQuantization | None, spec) -> bool:
    """Whether config.json has this tensor stored in 8-bit blocks."""
    return spec.block_scaled and quantization is not None and quantization.converts(spec.name)


def write_random_model(config: Mapping[str, Any], folder: str | Path, seed: int,
                       dtype: torch.dtype = torch.bfloat16) -> Path:
    """Write ``config.json`` and ``model.safetensors`` with seeded random weights."""
    from safetensors.torch import save_file
    folder = Path(folder)
    folder.mkdir(parents=True, exist_ok=True)
    config = dict(config)
    config["torch_dtype"] = str(dtype).replace("torch.", "")
    model = build_model(config, dtype=torch.float32, device="cpu")
    quantization = _quantization(config)
    tensors = {}
    for name, spec in model.expected_tensors().items():
        if spec.optional:
            continue  # e.g. a head tied to the embedding is not stored
        if _in_blocks(quantization, spec):
            matrix = quantize_matrix(random_tensor(spec, seed))
            tensors[name], tensors[name + SCALE_SUFFIX] = matrix.codes, matrix.scales
            continue
        tensors[name] = random_tensor(spec, seed, dtype=dtype).contiguous()
    (folder / "config.json").write_text(json.dumps(config, indent=1) + "\n")
    save_file(tensors, str(folder / SINGLE_FILE), metadata={"format": "pt", "seed": str(seed)})
    return folder


def init_random_weights(model, seed: int, storage_dtype: torch.dtype = torch.bfloat16, config: Mapping[str, Any] | None = None) -> None:
    """Bind seeded random weights generated on the model's device (nothing touches the disk).  ``config``: the config.json whose
    ``quantization_config`` says which matrices are stored in 8-bit blocks (None: none)."""
    quantization = None if config is None else _quantization(config)
    tensors = {}
    for name, spec in model.expected_tensors().items():
        if spec.optional:
            continue
        if _in_blocks(quantization, spec):
            tensors[name] = place_blocks(quantize_matrix(random_tensor(spec, seed, device=model.device)), model.dtype, model.device)
            continue
        raw = random_tensor(spec, seed, device=model.device, dtype=storage_dtype)
        tensors[name] = place(raw, spec.role, model.dtype, model.device)
    model.bind(tensors, consume=True)
