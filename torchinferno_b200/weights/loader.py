"""Weights from safetensors, bound by tensor name and checked against the model.

The reference reads tensors lazily by name through ``model.safetensors.index.json``
(src/torchinferno/models/llama3/pipeline.py:80-135) or from a lone
``model.safetensors`` (src/torchinferno/models/checkpoint_io.py:22-48), refuses
shard names that leave the folder (checkpoint_io.py:74-87) and does not compare
shapes with the configuration.  Here every name and shape is compared before
anything is copied, and one error lists all that is missing, unexpected or of
the wrong shape.

Storage rule: a tensor stored in bfloat16 stays bfloat16 and one stored in
32-bit stays 32-bit when the engine computes in bfloat16; norm vectors are
widened to fp32 (lossless); integer tables become int32.  When the engine
computes in float32 every floating tensor is widened to fp32.  A matrix that its
part takes in 8-bit blocks (``WeightSpec.block_scaled``) and that is stored as e4m3
codes with a tensor of scales beside it (its name and ``_scale_inv``) stays so in
bfloat16, and is widened to the numbers it stands for in float32; so does one stored as
4-bit codes with tensors of scales (its name and ``_scale``) and a factor (``_scale_2``)
beside it.  Codes without their scales are refused, and so are those of a folder whose
``quantization_config`` names other blocks, or another form of 4-bit codes (config/quantization.py).
"""
from __future__ import annotations

import json
from pathlib import Path
from typing import Iterable

import torch

from torchinferno_b200.config.model_config import ConfigError
from torchinferno_b200.config.quantization import (CODE_FACTOR_SUFFIX, CODE_SCALE_SUFFIX, SCALE_SUFFIX, BlockQuantization, check_codes,
                                                   measured_scale_of_rows, scales_of_a_cache)
from torchinferno_b200.kernels.block_scaled import BlockScaledMatrix, blocks
from torchinferno_b200.kernels.microscaled import RUN, MicroscaledMatrix

SINGLE_FILE = "model.safetensors"
INDEX_FILE = "model.safetensors.index.json"
CONFIG_FILE = "config.json"


class WeightError(ValueError):
    """The checkpoint does not hold what the model needs."""


# Buffers some exporters store beside the weights; they are recomputed from the configuration and never read.
# Anything else the model does not expect is an error.
IGNORED_SUFFIXES = ("rotary_emb.inv_freq", "self_attn.rotary_emb.inv_freq", "attn.masked_bias", "attn.bias")


_DTYPES = {"BF16": torch.bfloat16, "F32": torch.float32, "F16": torch.float16, "F64": torch.float64,
           "I32": torch.int32, "I64": torch.int64, "I16": torch.int16, "I8": torch.int8, "U8": torch.uint8,
           "BOOL": torch.bool}


def _safe_open(path: Path):
    from safetensors import safe_open
    return safe_open(str(path), framework="pt", device="cpu")


def checkpoint_files(folder: str | Path) -> dict[str, Path]:
    """Tensor name -> file that holds it."""
    folder = Path(folder)
    index = folder / INDEX_FILE
    single = folder / SINGLE_FILE
    if index.is_file():
        data = json.loads(index.read_text())
        weight_map = data.get("weight_map")
        if not isinstance(weight_map, dict):
            raise WeightError(f"{index} has no weight_map")
        root = folder.resolve()
        files: dict[str, Path] = {}
        for name, shard in weight_map.items():
            shard_path = (folder / str(shard)).resolve()
            if root not in shard_path.parents or not str(shard).endswith(".safetensors"):
                raise WeightError(f"{index}: shard {shard!r} of {name!r} is not a safetensors file inside the folder")
            if not shard_path.is_file():
                raise WeightError(f"{index}: shard {shard!r} of {name!r} does not exist")
            files[str(name)] = shard_path
        return files
    if single.is_file():
        with _safe_open(single) as handle:
            return {name: single for name in handle.keys()}
    raise FileNotFoundError(f"no {SINGLE_FILE} or {INDEX_FILE} in {folder}")


def _describe(names: Iterable[str], limit: int = 12) -> str:
    names = sorted(names)
    shown = ", ".join(names[:limit])
    return shown + (f", ... (+{len(names) - limit} more)" if len(names) > limit else "")


def load_weights(model, folder: str | Path) -> dict[str, object]:
    """Check the checkpoint against ``model.expected_tensors()``, copy it to the device and bind it."""
    files = checkpoint_files(folder)
    expected = model.expected_tensors()
    handles: dict[Path, object] = {}

    def handle_of(path: Path):
        if path not in handles:
            handles[path] = _safe_open(path).__enter__()
        return handles[path]

    try:
        missing = [n for n, ws in expected.items() if n not in files and not ws.optional]
        scales = {n + SCALE_SUFFIX: n for n, ws in expected.items() if ws.block_scaled and n in files}
        in_blocks = {n for s, n in scales.items() if s in files}
        in_codes = {n for n, ws in expected.items() if ws.block_scaled and n in files and n + CODE_SCALE_SUFFIX in files and n + CODE_FACTOR_SUFFIX in files}
        beside_codes = {n + suffix for n in in_codes for suffix in (CODE_SCALE_SUFFIX, CODE_FACTOR_SUFFIX)}
        not_needed = {measured_scale_of_rows(n) for n in in_codes}
        if in_codes:      # (whichever of the matrices are in codes)
            not_needed.update(scale for n, ws in expected.items() if ws.block_scaled for scale in scales_of_a_cache(n))
        ignored = sorted(n for n in files if n not in expected and (n.endswith(IGNORED_SUFFIXES) or n in not_needed))
        unexpected = [n for n in files if n not in expected and n not in ignored and scales.get(n) not in in_blocks and n not in beside_codes]
        # a head that the model ties to its embedding is not read even if the file stores a copy
        unused = set(model.unused_optional_tensors()) if hasattr(model, "unused_optional_tensors") else set()
        wrong: list[str] = []
        for name, ws in expected.items():
            if name not in files:
                continue
            view = handle_of(files[name]).get_slice(name)
            shape = tuple(view.get_shape())
            if name in in_codes:
                wrong += _wrong_codes(name, ws.shape, *(handle_of(files[n]).get_slice(n) for n in (name, name + CODE_SCALE_SUFFIX, name + CODE_FACTOR_SUFFIX)))
                continue
            free = getattr(ws, "free_dims", ())
            if len(shape) != len(ws.shape) or any(a != b for d, (a, b) in enumerate(zip(shape, ws.shape)) if d not in free):
                wrong.append(f"{name}: file {list(shape)} vs model {list(ws.shape)}")
            dtype = str(view.get_dtype())
            if name in in_blocks:
                beside = handle_of(files[name + SCALE_SUFFIX]).get_slice(name + SCALE_SUFFIX)
                found = list(beside.get_shape())
                if found != [blocks(d) for d in shape]:
                    wrong.append(f"{name + SCALE_SUFFIX}: file {found} vs a scale for each 128 x 128 of {list(shape)}")
                elif dtype != "F8_E4M3":
                    wrong.append(f"{name}: has scales beside it but is not stored as e4m3 codes")
                elif not str(beside.get_dtype()).startswith(("F", "BF")):
                    wrong.append(f"{name + SCALE_SUFFIX}: stored as {beside.get_dtype()}, scales are floating-point numbers")
            elif dtype.startswith("F8") and name not in unused:      # (codes stand for nothing without their scales)
                wrong.append(f"{name}: stored as {dtype} without {name + SCALE_SUFFIX}" if ws.block_scaled else f"{name}: stored as {dtype}, which the model does not take")
            elif dtype == "U8" and ws.block_scaled:
                wrong.append(f"{name}: stored as {dtype} without {name + CODE_SCALE_SUFFIX} and {name + CODE_FACTOR_SUFFIX}")
        if missing or unexpected or wrong:
            parts = [f"checkpoint {folder} does not fit the model ({model.spec.architecture}):"]
            if missing:
                parts.append(f"  missing ({len(missing)}): {_describe(missing)}")
            if unexpected:
                parts.append(f"  unexpected ({len(unexpected)}): {_describe(unexpected)}")
            if wrong:
                parts.append(f"  wrong shape ({len(wrong)}): " + "; ".join(sorted(wrong)[:12])
                             + (f"; ... (+{len(wrong) - 12} more)" if len(wrong) > 12 else ""))
            raise WeightError("\n".join(parts))
        if (in_blocks or in_codes) and (Path(folder) / CONFIG_FILE).is_file():
            said = json.loads((Path(folder) / CONFIG_FILE).read_text())
            for held, check, what in ((in_blocks, BlockQuantization.from_config, "8-bit blocks"), (in_codes, check_codes, "4-bit codes")):
                try:
                    if held:
                        check(said)
                except ConfigError as exc:
                    raise WeightError(f"checkpoint {folder} holds {what}, but {exc}") from None
        tensors: dict[str, torch.Tensor] = {}
        stored: dict[str, str] = {}
        for name, ws in expected.items():
            if name not in files or name in unused:
                continue
            tensor = handle_of(files[name]).get_tensor(name)
            stored[name] = str(tensor.dtype).replace("torch.", "")
            if name in in_blocks:
                matrix = BlockScaledMatrix(tensor.contiguous(), handle_of(files[name + SCALE_SUFFIX]).get_tensor(name + SCALE_SUFFIX).to(torch.float32).contiguous())
                tensors[name] = place_blocks(matrix, model.dtype, model.device)
            elif name in in_codes:
                beside, factor = (handle_of(files[name + suffix]).get_tensor(name + suffix) for suffix in (CODE_SCALE_SUFFIX, CODE_FACTOR_SUFFIX))
                matrix = MicroscaledMatrix(tensor.contiguous(), beside.contiguous(), factor.to(torch.float32).reshape(()), ws.shape[1])
                tensors[name] = place_blocks(matrix, model.dtype, model.device)
            else:
                tensors[name] = place(tensor, ws.role, model.dtype, model.device)
    finally:
        for handle in handles.values():
            handle.__exit__(None, None, None)
    count = len(tensors)
    model.bind(tensors, consume=True)      # (each part's source tensors are dropped as it binds them)
    return {"tensors": count, "stored_dtypes": sorted(set(stored.values())), "ignored": ignored,
            "not_read": sorted(unused & set(files))}


def _wrong_codes(name: str, wanted: tuple[int, ...], codes, scales, factor) -> list[str]:
    """What does not fit of a matrix of 4-bit codes and the tensors beside it (slices of the file)."""
    n, k = wanted
    found = {name: codes, name + CODE_SCALE_SUFFIX: scales, name + CODE_FACTOR_SUFFIX: factor}
    shapes = {name: [[n, -(-k // 2)]], name + CODE_SCALE_SUFFIX: [[n, -(-k // RUN)]], name + CODE_FACTOR_SUFFIX: [[], [1]]}
    kinds = {name: "U8", name + CODE_SCALE_SUFFIX: "F8_E4M3", name + CODE_FACTOR_SUFFIX: "F32"}
    wrong = [f"{t}: file {list(view.get_shape())} vs {shapes[t][0]} of a 4-bit {list(wanted)}" for t, view in found.items() if list(view.get_shape()) not in shapes[t]]
    return wrong + [f"{t}: stored as {view.get_dtype()}, of a matrix of 4-bit codes it is {kinds[t]}" for t, view in found.items() if str(view.get_dtype()) != kinds[t]]


def place_blocks(matrix: "BlockScaledMatrix | MicroscaledMatrix", compute_dtype: torch.dtype, device: torch.device) -> "BlockScaledMatrix | MicroscaledMatrix | torch.Tensor":
    """The same for a matrix in 8-bit blocks or 4-bit codes."""
    matrix = matrix.to(device)
    return matrix.widened(torch.float32) if compute_dtype == torch.float32 else matrix


def place(tensor: torch.Tensor, role: str, compute_dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """Apply the storage rule to one tensor and move it to the device."""
    if role == "int_table" or not tensor.is_floating_point():
        return tensor.to(torch.int32).contiguous().to(device)
    if role == "vector" or compute_dtype == torch.float32:
        return tensor.to(torch.float32).contiguous().to(device)
    if tensor.dtype in (torch.bfloat16, torch.float32):
        return tensor.contiguous().to(device)
    return tensor.to(torch.bfloat16).contiguous().to(device)
