"""``quantization_config`` of a ``config.json``: which tensors a checkpoint stores in 8 bits, and how.

One form is read, ``"quant_method": "fp8"`` with a scale for each block of 128 x 128 (``"weight_block_size": [128, 128]``): a matrix ``name`` is e4m3
codes, its scales are the 32-bit tensor ``name + "_scale_inv"``, and activations are quantised as they come (``"activation_scheme": "dynamic"``).
The rows' scales are powers of two (kernels/block_scaled.py), whether or not the file says so (``scale_fmt``).
Which of a model's matrices may be stored so is up to its parts (``WeightSpec.block_scaled``); which of them are is seen from the file.
Other methods are left to the loader, which refuses tensors that the model does not know; a file with 8-bit blocks is checked against this form, and random
models leave any other aside.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Any, Mapping

from torchinferno_b200.config.model_config import ConfigError

SCALE_SUFFIX = "_scale_inv"


@dataclass(frozen=True)
class BlockQuantization:
    """8-bit blocks for every matrix that may have them, but for the modules named here."""
    not_converted: tuple[str, ...] = ()

    @classmethod
    def from_config(cls, config: Mapping[str, Any]) -> "BlockQuantization | None":
        data = config.get("quantization_config")
        if data is None:
            return None
        if not isinstance(data, Mapping):
            raise ConfigError(f"quantization_config must be an object or null, got {type(data).__name__}")
        if str(data.get("quant_method", "")).lower() != "fp8":
            return None
        block = data.get("weight_block_size")
        if not isinstance(block, (list, tuple)) or list(block) != [128, 128]:
            raise ConfigError(f"quantization_config.weight_block_size={block!r} is not supported (fp8 weights have a scale for each block of [128, 128])")
        if str(data.get("fmt", "e4m3")).lower() != "e4m3":
            raise ConfigError(f"quantization_config.fmt={data['fmt']!r} is not supported (e4m3)")
        if str(data.get("activation_scheme", "dynamic")).lower() != "dynamic":
            raise ConfigError(f"quantization_config.activation_scheme={data['activation_scheme']!r} is not supported (dynamic)")
        names = data.get("modules_to_not_convert") or data.get("ignored_layers") or ()
        if not isinstance(names, (list, tuple)) or not all(isinstance(n, str) for n in names):
            raise ConfigError("quantization_config.modules_to_not_convert must be a list of names")
        return cls(tuple(names))

    def converts(self, name: str) -> bool:
        """Whether the tensor ``name`` is outside the modules that stay as they are (named in full, by a prefix or by a part of their path)."""
        return not any(f".{module}." in f".{name}." for module in self.not_converted)
