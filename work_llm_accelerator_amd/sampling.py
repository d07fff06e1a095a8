"""Token sampling from logits (include/qwen_hip_sample.h) driven from Python.

The reference only takes the argmax (verification/qwen_full_model_validation.py:128,159; `DeviceModel.greedy`).
The random numbers are the caller's, so a draw can be repeated.  Every value is computed by the HIP library on the
current stream of the logits' device; nothing is synchronized.
"""

from __future__ import annotations

import ctypes

import torch

from . import abi
from .kv8 import MAX_COUNT, _check, _on, _raw_stream, _type_of


def row_params(rows: int, device, uniforms, temperature, top_k, top_p, min_p, token_ids) -> list:
    """Pointers of the per-row arguments (None stays null), checked: contiguous [rows] on `device`, float32, top_k
    and token_ids int32."""
    out = []
    for name, t, dtype in (("uniforms", uniforms, torch.float32), ("temperature", temperature, torch.float32),
                           ("top_k", top_k, torch.int32), ("top_p", top_p, torch.float32),
                           ("min_p", min_p, torch.float32), ("token_ids", token_ids, torch.int32)):
        if t is None and name not in ("uniforms", "token_ids"):
            out.append(None)
            continue
        if t.dtype != dtype or t.shape != (rows,) or not t.is_contiguous() or t.device != device:
            raise ValueError(f"{name} must be {rows} contiguous {dtype} values on {device}")
        out.append(t.data_ptr())
    return out


def sample_logits(logits, uniforms, temperature=None, top_k=None, top_p=None, min_p=None, token_ids=None):
    """One token per row of logits [rows, vocab] (float32 or bfloat16, rows contiguous): temperature, then top-k,
    top-p over what top-k keeps, min-p, and the draw by uniforms [rows] in [0, 1).  temperature, top_p, min_p [rows]
    float32 and top_k [rows] int32 on the GPU, None for off (temperature 1); a temperature of 0 takes the
    argmax.  Returns token_ids [rows] int32 (a new tensor unless given)."""
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("logits must be [rows, vocab] with contiguous rows")
    rows, vocab = logits.shape
    if rows > MAX_COUNT or vocab > MAX_COUNT:
        raise ValueError(f"logits must be at most {MAX_COUNT} each way")
    if token_ids is None:
        token_ids = torch.empty(rows, dtype=torch.int32, device=logits.device)
    kind, lib = _type_of(logits), abi.load()
    u, t, k, p, q, ids = row_params(rows, logits.device, uniforms, temperature, top_k, top_p, min_p, token_ids)
    need = ctypes.c_uint64(0)
    with _on(logits.device):
        _check(lib, lib.qwen_hip_sample_workspace(rows, vocab, ctypes.byref(need)), "qwen_hip_sample_workspace")
        ws = torch.empty(need.value, dtype=torch.uint8, device=logits.device) if need.value else None
        st = lib.qwen_hip_sample(logits.data_ptr(), kind, logits.stride(0), rows, vocab, u, t, k, p, q, ids,
                                 ws.data_ptr() if ws is not None else None, need.value,
                                 _raw_stream(logits.device.index))
    _check(lib, st, "qwen_hip_sample")
    return token_ids


__all__ = ["sample_logits"]
