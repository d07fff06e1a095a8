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
from dataclasses import dataclass

from . import abi
from .layout import HEAD_DIM, KV_HEADS

BLOCK = 64  # tokens that share a scale
TYPE_F32 = 0
TYPE_BF16 = 1
ZERO_OUTSIDE = 0x1


def _check(lib, status: int, what: str) -> None:
    if status == 1:
        raise ValueError(f"{what}: {abi.last_error(lib)}")
    if status != 0:
        raise RuntimeError(f"{what} failed with status {status}: {abi.last_error(lib)}")


def _type_of(t) -> int:
    import torch

    if t.dtype == torch.float32:
        return TYPE_F32
    if t.dtype == torch.bfloat16:
        return TYPE_BF16
    raise ValueError(f"rows must be float32 or bfloat16, not {t.dtype}")


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
        import torch

        if self.k.dim() != 5 or self.k.shape[4] % BLOCK != 0:
            raise ValueError("codes must be [layers, sequences, blocks, kv_heads, 64 * head_dim]")
        for t, shape, dtype in ((self.k, self.k.shape, torch.int8), (self.v, self.k.shape, torch.int8),
                                (self.k_scale, self.k.shape[:4], torch.float32),
                                (self.v_scale, self.k.shape[:4], torch.float32)):
            if t.shape != shape or t.dtype != dtype or not t.is_contiguous() or t.device != self.k.device:
                raise ValueError("codes (int8) and scales (float32) must be contiguous, on one device and of one cache shape")

    @classmethod
    def allocate(cls, layers: int, sequences: int, positions: int, kv_heads: int = KV_HEADS,
                 head_dim: int = HEAD_DIM, device="cuda:0"):
        """An empty cache of at least `positions` tokens a sequence (whole blocks)."""
        import torch

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
        if not 0 <= layer < self.layers:
            raise ValueError(f"layer {layer} of {self.layers}")
        sequences, blocks, heads, width = self.k.shape[1:]
        n = sequences * blocks * heads
        return abi.Kv8CacheStruct(self.k.data_ptr() + layer * n * width, self.v.data_ptr() + layer * n * width,
                                  self.k_scale.data_ptr() + 4 * layer * n, self.v_scale.data_ptr() + 4 * layer * n,
                                  sequences, blocks, heads, width // BLOCK)

    def _rows(self, t, batch: int, rows: int, heads: int, what: str) -> abi.Kv8RowsStruct:
        if tuple(t.shape) != (batch, rows, heads, self.head_dim):
            raise ValueError(f"{what} must be {(batch, rows, heads, self.head_dim)}, not {tuple(t.shape)}")
        if t.device != self.k.device:
            raise ValueError(f"{what} must be on {self.k.device}, not {t.device}")
        if t.stride(3) != 1:
            raise ValueError(f"{what}: the values of a row must be contiguous")
        return abi.Kv8RowsStruct(t.data_ptr(), t.stride(0), t.stride(1), t.stride(2))

    def _positions(self, positions, batch: int):
        import torch

        if positions.dtype != torch.int32 or tuple(positions.shape) != (batch,) or not positions.is_contiguous():
            raise ValueError(f"positions must be {batch} contiguous int32 values")
        if positions.device != self.k.device:
            raise ValueError(f"positions must be on {self.k.device}, not {positions.device}")
        return ctypes.c_void_p(positions.data_ptr())

    def _stream(self):
        import torch

        return ctypes.c_void_p(torch.cuda.current_stream(self.k.device).cuda_stream)

    def store(self, layer: int, k, v, positions) -> None:
        """Stores k, v [batch, rows, kv_heads, head_dim] (float32 or bfloat16, any strides of whole 16 bytes) as
        tokens positions[b] .. positions[b] + rows - 1 of sequences 0..batch-1; positions [batch] int32 on the
        GPU.  A negative position leaves its sequence as it is; tokens behind the cache are dropped."""
        import torch

        if k.dim() != 4:
            raise ValueError("k must be [batch, rows, kv_heads, head_dim]")
        if k.dtype != v.dtype:
            raise ValueError("k and v must have one type")
        batch, rows = k.shape[:2]
        ks, vs = self._rows(k, batch, rows, self.kv_heads, "k"), self._rows(v, batch, rows, self.kv_heads, "v")
        pos, c, lib = self._positions(positions, batch), self.layer_struct(layer), abi.load()
        with torch.cuda.device(self.k.device):
            st = lib.qwen_hip_kv8_store(ctypes.byref(c), _type_of(k), ctypes.byref(ks), ctypes.byref(vs), batch, rows,
                                        pos, self._stream())
        _check(lib, st, "qwen_hip_kv8_store")

    def load(self, layer: int, positions, rows: int | None = None, k=None, v=None, dtype=None):
        """Tokens positions[b] .. positions[b] + rows - 1 as rows (k, v) [batch, rows, kv_heads, head_dim]: into the
        tensors given (rows of tokens outside the cache are left as they are), or into new ones of `dtype`
        (float32 by default; rows outside the cache are zeros)."""
        import torch

        if (k is None) != (v is None):
            raise ValueError("k and v are given together")
        flags = 0
        if k is None:
            if rows is None:
                raise ValueError("rows is needed where no tensors are given")
            shape = (positions.shape[0], rows, self.kv_heads, self.head_dim)
            k, v = (torch.empty(shape, dtype=dtype or torch.float32, device=self.k.device) for _ in range(2))
            flags = ZERO_OUTSIDE
        elif k.dim() != 4 or (rows is not None and rows != k.shape[1]) or (dtype is not None and dtype != k.dtype):
            raise ValueError("k and v must be [batch, rows, kv_heads, head_dim] of the rows and type asked for")
        if k.dtype != v.dtype:
            raise ValueError("k and v must have one type")
        batch, rows = k.shape[:2]
        ks, vs = self._rows(k, batch, rows, self.kv_heads, "k"), self._rows(v, batch, rows, self.kv_heads, "v")
        pos, c, lib = self._positions(positions, batch), self.layer_struct(layer), abi.load()
        with torch.cuda.device(self.k.device):
            st = lib.qwen_hip_kv8_load(ctypes.byref(c), _type_of(k), ctypes.byref(ks), ctypes.byref(vs), batch, rows,
                                       flags, pos, self._stream())
        _check(lib, st, "qwen_hip_kv8_load")
        return k, v

    def attend(self, layer: int, q, positions, max_keys: int, out=None, scale: float | None = None):
        """Causal attention of q [batch, rows, q_heads, head_dim] (float32 or bfloat16) over the cache, whose own
        K/V rows are stored already: query i of sequence b attends tokens 0 .. positions[b] + i; a query with
        none gives zeros.  max_keys: at least max(positions) + rows.  scale: 1 / sqrt(head_dim) by default.
        Returns out (a new tensor unless given)."""
        import torch

        if q.dim() != 4:
            raise ValueError("q must be [batch, rows, q_heads, head_dim]")
        batch, rows, heads = q.shape[:3]
        if out is None:
            out = torch.empty((batch, rows, heads, self.head_dim), dtype=q.dtype, device=q.device)
        if out.dtype != q.dtype:
            raise ValueError("q and out must have one type")
        qs, os = self._rows(q, batch, rows, heads, "q"), self._rows(out, batch, rows, heads, "out")
        pos, c, lib, kind = self._positions(positions, batch), self.layer_struct(layer), abi.load(), _type_of(q)
        need = ctypes.c_uint64(0)
        with torch.cuda.device(self.k.device):
            _check(lib, lib.qwen_hip_kv8_attention_workspace(ctypes.byref(c), kind, heads, batch, rows, int(max_keys),
                                                             ctypes.byref(need)), "qwen_hip_kv8_attention_workspace")
            # the stream's own allocation: reused by later work of this stream only, private to a graph being captured
            ws = torch.empty(need.value, dtype=torch.uint8, device=self.k.device) if need.value else None
            st = lib.qwen_hip_kv8_attention(ctypes.byref(c), kind, ctypes.byref(qs), ctypes.byref(os), heads, batch, rows,
                                            pos, int(max_keys), 1.0 / math.sqrt(self.head_dim) if scale is None else scale,
                                            ctypes.c_void_p(ws.data_ptr()) if ws is not None else None, need.value,
                                            self._stream())
        _check(lib, st, "qwen_hip_kv8_attention")
        return out


__all__ = ["Kv8Cache", "BLOCK"]
