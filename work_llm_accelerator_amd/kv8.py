"""K/V cache in 8 bits and the attention over it (include/qwen_hip_kv8.h) driven from Python.

The reference keeps fp32 caches only (hls/common/llm_memory_layout.h:130-149); `Kv8Cache` is the compact form
beside `model.KvCache`: int8 codes with one power-of-two scale per 64 tokens, KV head and K or V.  torch owns the
memory; every value is computed by the HIP library on the current stream of the cache's device.  Nothing is
synchronized, so the calls can be captured into a graph; calls on different streams that share a cache are the
caller's to order.
"""

from __future__ import annotations

import ctypes
import math
from contextlib import nullcontext
from dataclasses import dataclass

import torch

from . import abi
from .layout import HEAD_DIM, KV_HEADS

BLOCK = 64  # tokens that share a scale
TYPE_F32 = 0
TYPE_BF16 = 1
ZERO_OUTSIDE = 0x1
MAX_COUNT = 1 << 24


def _check(lib, status: int, what: str) -> None:
    if status == 1:
        raise ValueError(f"{what}: {abi.last_error(lib)}")
    if status != 0:
        raise RuntimeError(f"{what} failed with status {status}: {abi.last_error(lib)}")


_TYPES = {torch.float32: TYPE_F32, torch.bfloat16: TYPE_BF16}


def _type_of(t) -> int:
    kind = _TYPES.get(t.dtype)
    if kind is None:
        raise ValueError(f"rows must be float32 or bfloat16, not {t.dtype}")
    return kind


# The raw stream of a device; torch.cuda.current_stream() makes a Stream object first, which takes longer than
# the rest of a call's checks (1.8 us).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_HERE = nullcontext()


def _on(device):
    """A context in which `device` is the current one."""
    return _HERE if _current_device() == device.index else torch.cuda.device(device)


@dataclass
class Kv8Cache:
    """Codes [layers][sequences][blocks][kv_heads][64 * head_dim] int8 and scales [layers][sequences][blocks]
    [kv_heads] fp32 of K and V, contiguous, on one GPU; the order of the codes within a block is described in
    include/qwen_hip_kv8.h."""

    k: "object"  # torch.Tensor on the GPU
    v: "object"
    k_scale: "object"
    v_scale: "object"

    def __post_init__(self):
        k, v, shape, device = self.k, self.v, self.k.shape, self.k.device
        if len(shape) != 5 or shape[4] % BLOCK != 0:
            raise ValueError("codes must be [layers, sequences, blocks, kv_heads, 64 * head_dim]")
        ks, vs, scales = self.k_scale, self.v_scale, shape[:4]
        if (v.shape != shape or ks.shape != scales or vs.shape != scales or k.dtype != torch.int8 or v.dtype != torch.int8
                or ks.dtype != torch.float32 or vs.dtype != torch.float32 or v.device != device or ks.device != device
                or vs.device != device
                or not (k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous())):
            raise ValueError("codes (int8) and scales (float32) must be contiguous, on one device and of one cache shape")

    @classmethod
    def allocate(cls, layers: int, sequences: int, positions: int, kv_heads: int = KV_HEADS,
                 head_dim: int = HEAD_DIM, device="cuda:0"):
        """An empty cache of at least `positions` tokens a sequence (whole blocks)."""
        shape = (layers, sequences, (positions + BLOCK - 1) // BLOCK, kv_heads)
        return cls(*(torch.zeros((*shape, BLOCK * head_dim), dtype=torch.int8, device=device) for _ in range(2)),
                   *(torch.zeros(shape, dtype=torch.float32, device=device) for _ in range(2)))

    @property
    def layers(self) -> int:
        return self.k.shape[0]

    @property
    def sequences(self) -> int:
        return self.k.shape[1]

    @property
    def positions(self) -> int:
        """Tokens that a sequence can hold."""
        return self.k.shape[2] * BLOCK

    @property
    def kv_heads(self) -> int:
        return self.k.shape[3]

    @property
    def head_dim(self) -> int:
        return self.k.shape[4] // BLOCK

    def layer_struct(self, layer: int) -> abi.Kv8CacheStruct:
        layers, sequences, blocks, heads, width = self.k.shape
        if not 0 <= layer < layers:
            raise ValueError(f"layer {layer} of {layers}")
        n = layer * sequences * blocks * heads
        return abi.Kv8CacheStruct(self.k.data_ptr() + n * width, self.v.data_ptr() + n * width,
                                  self.k_scale.data_ptr() + 4 * n, self.v_scale.data_ptr() + 4 * n, sequences, blocks,
                                  heads, width // BLOCK)

    def _rows(self, t, shape: tuple, device, what: str) -> abi.Kv8RowsStruct:
        """`t` of `shape` on `device` as qwen_kv8_rows."""
        strides = t.stride()
        if t.shape != shape:
            raise ValueError(f"{what} must be {shape}, not {tuple(t.shape)}")
        if max(shape) > MAX_COUNT:  # (ctypes would cut it to 32 bits)
            raise ValueError(f"{what} has a dimension above {MAX_COUNT}")
        if t.device != device:
            raise ValueError(f"{what} must be on {device}, not {t.device}")
        if strides[3] != 1:
            raise ValueError(f"{what}: the values of a row must be contiguous")
        return abi.Kv8RowsStruct(t.data_ptr(), strides[0], strides[1], strides[2])

    def _positions(self, positions, batch: int, device) -> int:
        if positions.dtype != torch.int32 or positions.shape != (batch,) or not positions.is_contiguous():
            raise ValueError(f"positions must be {batch} contiguous int32 values")
        if positions.device != device:
            raise ValueError(f"positions must be on {device}, not {positions.device}")
        return positions.data_ptr()

    def store(self, layer: int, k, v, positions) -> None:
        """Stores k, v [batch, rows, kv_heads, head_dim] (float32 or bfloat16, any strides of whole 16 bytes) as
        tokens positions[b] .. positions[b] + rows - 1 of sequences 0..batch-1; positions [batch] int32 on the
        GPU.  A negative position leaves its sequence as it is; tokens behind the cache are dropped."""
        if k.dim() != 4:
            raise ValueError("k must be [batch, rows, kv_heads, head_dim]")
        if k.dtype != v.dtype:
            raise ValueError("k and v must have one type")
        batch, rows = k.shape[:2]
        c, lib, device = self.layer_struct(layer), abi.load(), self.k.device
        shape = (batch, rows, c.kv_heads, c.head_dim)
        ks, vs = self._rows(k, shape, device, "k"), self._rows(v, shape, device, "v")
        pos = self._positions(positions, batch, device)
        with _on(device):
            st = lib.qwen_hip_kv8_store(ctypes.byref(c), _type_of(k), ctypes.byref(ks), ctypes.byref(vs), batch, rows,
                                        pos, _raw_stream(device.index))
        _check(lib, st, "qwen_hip_kv8_store")

    def load(self, layer: int, positions, rows: int | None = None, k=None, v=None, dtype=None):
        """Tokens positions[b] .. positions[b] + rows - 1 as rows (k, v) [batch, rows, kv_heads, head_dim]: into the
        tensors given (rows of tokens outside the cache are left as they are), or into new ones of `dtype`
        (float32 by default; rows outside the cache are zeros)."""
        if (k is None) != (v is None):
            raise ValueError("k and v are given together")
        flags = 0
        if k is None:
            if rows is None:
                raise ValueError("rows is needed where no tensors are given")
            shape = (positions.shape[0], rows, self.kv_heads, self.head_dim)
            k, v = torch.empty((2, *shape), dtype=dtype or torch.float32, device=self.k.device).unbind()
            flags = ZERO_OUTSIDE
        elif k.dim() != 4 or (rows is not None and rows != k.shape[1]) or (dtype is not None and dtype != k.dtype):
            raise ValueError("k and v must be [batch, rows, kv_heads, head_dim] of the rows and type asked for")
        if k.dtype != v.dtype:
            raise ValueError("k and v must have one type")
        batch, rows = k.shape[:2]
        c, lib, device = self.layer_struct(layer), abi.load(), self.k.device
        shape = (batch, rows, c.kv_heads, c.head_dim)
        ks, vs = self._rows(k, shape, device, "k"), self._rows(v, shape, device, "v")
        pos = self._positions(positions, batch, device)
        with _on(device):
            st = lib.qwen_hip_kv8_load(ctypes.byref(c), _type_of(k), ctypes.byref(ks), ctypes.byref(vs), batch, rows,
                                       flags, pos, _raw_stream(device.index))
        _check(lib, st, "qwen_hip_kv8_load")
        return k, v

    def attend(self, layer: int, q, positions, max_keys: int, out=None, scale: float | None = None):
        """Causal attention of q [batch, rows, q_heads, head_dim] (float32 or bfloat16) over the cache, whose own
        K/V rows are stored already: query i of sequence b attends tokens 0 .. positions[b] + i; a query with
        none gives zeros.  max_keys: at least max(positions) + rows.  scale: 1 / sqrt(head_dim) by default.
        Returns out (a new tensor unless given)."""
        if q.dim() != 4:
            raise ValueError("q must be [batch, rows, q_heads, head_dim]")
        batch, rows, heads = q.shape[:3]
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        if out.dtype != q.dtype:
            raise ValueError("q and out must have one type")
        max_keys, c, lib, kind, device = int(max_keys), self.layer_struct(layer), abi.load(), _type_of(q), self.k.device
        if not 0 < max_keys <= BLOCK * c.blocks:
            raise ValueError(f"max_keys must be 1 .. {BLOCK * c.blocks}, not {max_keys}")
        shape = (batch, rows, heads, c.head_dim)
        qs, os = self._rows(q, shape, device, "q"), self._rows(out, shape, device, "out")
        pos = self._positions(positions, batch, device)
        need = ctypes.c_uint64(0)
        with _on(device):
            _check(lib, lib.qwen_hip_kv8_attention_workspace(ctypes.byref(c), kind, heads, batch, rows, max_keys,
                                                             ctypes.byref(need)), "qwen_hip_kv8_attention_workspace")
            # the stream's own allocation: reused by later work of this stream only, private to a graph being captured
            ws = torch.empty(need.value, dtype=torch.uint8, device=device) if need.value else None
            st = lib.qwen_hip_kv8_attention(ctypes.byref(c), kind, ctypes.byref(qs), ctypes.byref(os), heads, batch, rows,
                                            pos, max_keys, 1.0 / math.sqrt(self.head_dim) if scale is None else scale,
                                            ws.data_ptr() if ws is not None else None, need.value,
                                            _raw_stream(device.index))
        _check(lib, st, "qwen_hip_kv8_attention")
        return out


__all__ = ["Kv8Cache", "BLOCK"]
