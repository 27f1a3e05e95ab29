"""``quantization_config`` of a ``config.json``: which tensors a checkpoint stores in 8 or 4 bits, and how.

Two forms are read.  ``"quant_method": "fp8"`` with a scale for each block of 128 x 128 (``"weight_block_size": [128, 128]``): a matrix ``name`` is e4m3
codes, its scales are the 32-bit tensor ``name + "_scale_inv"``, and activations are quantised as they come (``"activation_scheme": "dynamic"``).
The rows' scales are powers of two (kernels/block_scaled.py), whether or not the file says so (``scale_fmt``).
``"quant_algo": "NVFP4"``: a matrix ``name`` is e2m1 codes, two in a byte, with an e4m3 scale for each 16 columns (``name + "_scale"``) and one 32-bit factor
(``name + "_scale_2"``); the rows' scales are their own (kernels/microscaled.py), so the measured ones that such files hold (``input_scale``), and those of an
8-bit cache (``k_scale``, ``v_scale``), are not read.
Which of a model's matrices may be stored so is up to its parts (``WeightSpec.block_scaled``); which of them are is seen from the file.
Other methods are left to the loader, which refuses tensors that the model does not know; a file with 8-bit blocks or 4-bit codes is checked against its form, and random
models leave any other aside.
"""
from __future__ import annotations

from dataclasses import dataclass
from fnmatch import fnmatchcase
from typing import Any, Mapping

from torchinferno_b200.config.model_config import ConfigError

SCALE_SUFFIX = "_scale_inv"
CODE_SCALE_SUFFIX, CODE_FACTOR_SUFFIX = "_scale", "_scale_2"


def measured_scale_of_rows(name: str) -> str | None:
    """The tensor that files in 4 bits hold beside the matrix ``name`` for the rows it meets, which is not read."""
    return name.removesuffix("weight") + "input_scale" if name.endswith(".weight") else None


def scales_of_a_cache(name: str) -> tuple[str, ...]:
    """The tensors that files in 4 bits which were made for a key and value cache in 8 bits hold beside the projection ``name``.  They concern such a cache alone, and
    are not read: the cache here has the model's own type."""
    return tuple(name.removesuffix("weight") + suffix for suffix in ("k_scale", "v_scale")) if name.endswith(".weight") else ()


def _settings(config: Mapping[str, Any]) -> Mapping[str, Any]:
    data = config.get("quantization_config")
    if data is not None and not isinstance(data, Mapping):
        raise ConfigError(f"quantization_config must be an object or null, got {type(data).__name__}")
    return data or {}


@dataclass(frozen=True)
class BlockQuantization:
    """8-bit blocks for every matrix that may have them, but for the modules named here."""
    not_converted: tuple[str, ...] = ()

    @classmethod
    def from_config(cls, config: Mapping[str, Any]) -> "BlockQuantization | None":
        data = _settings(config)
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


@dataclass(frozen=True)
class MicroscaledQuantization:
    """4-bit codes for every matrix that may have them, but for the modules named here (names, or patterns with ``*``)."""
    ignored: tuple[str, ...] = ()

    @classmethod
    def from_config(cls, config: Mapping[str, Any]) -> "MicroscaledQuantization | None":
        data = _settings(config)
        if str(data.get("quant_algo", "")).upper() != "NVFP4":
            return None
        groups = data.get("config_groups") or {}
        sizes = [data.get("group_size")]
        if not isinstance(groups, Mapping):
            raise ConfigError("quantization_config.config_groups must be an object")
        for group in groups.values():
            weights = group.get("weights") if isinstance(group, Mapping) else None
            sizes.append(weights.get("group_size") if isinstance(weights, Mapping) else None)
        if any(size not in (None, 16) for size in sizes):
            raise ConfigError(f"quantization_config: groups of {[s for s in sizes if s is not None]} columns are not supported (4-bit codes have a scale for each 16)")
        names = data.get("ignore") or data.get("exclude_modules") or ()
        if not isinstance(names, (list, tuple)) or not all(isinstance(n, str) for n in names):
            raise ConfigError("quantization_config.ignore must be a list of names")
        return cls(tuple(names))

    def converts(self, name: str) -> bool:
        """Whether the tensor ``name`` is outside the modules that stay as they are (named in full, by a prefix, by a part of their path or by a pattern)."""
        return not any(f".{module}." in f".{name}." or fnmatchcase(name, module) or fnmatchcase(name.rpartition(".")[0], module) for module in self.ignored)


def check_codes(config: Mapping[str, Any]) -> None:
    """Raises ConfigError where config.json says of a folder that holds 4-bit codes that they are of another form.  (One that says nothing of them is taken by its tensors.)"""
    data = _settings(config)
    algo, method = (str(data.get(key) or "") for key in ("quant_algo", "quant_method"))
    if algo.upper() not in ("", "NVFP4") or (not algo and method and not method.lower().startswith("modelopt")):
        raise ConfigError(f"quantization_config names {algo or method!r} (codes with a scale for each 16 columns are 'NVFP4')")
    MicroscaledQuantization.from_config(config)


def quantization_of(config: Mapping[str, Any]) -> "BlockQuantization | MicroscaledQuantization | None":
    """The form of quantised weights that config.json names, if it is one that is read."""
    return BlockQuantization.from_config(config) or MicroscaledQuantization.from_config(config)
