"""Arguments that the 8-bit cache and the sampling entry points refuse, before anything reaches a GPU."""

from __future__ import annotations

import ctypes

import pytest

from work_llm_accelerator_amd import abi

PTR = 1 << 20  # aligned, never read: every call here is refused


@pytest.fixture(scope="module")
def lib():
    return abi.load()


def cache(**over):
    f = dict(k=PTR, v=PTR, k_scale=PTR, v_scale=PTR, sequences=4, blocks=8, kv_heads=2, head_dim=128)
    f.update(over)
    return abi.Kv8CacheStruct(*f.values())


def rows(data=PTR, seq=1 << 20, token=256, head=128):
    return abi.Kv8RowsStruct(data, seq, token, head)


def call(lib, op, c=None, kind=0, a=None, b=None, batch=2, n=3, positions=PTR, heads=4, max_keys=64, scale=0.1, flags=0,
         ws=PTR, ws_bytes=1 << 40):
    c = cache() if c is None else c
    a, b = a or rows(token=512), b or rows(token=512)
    c, a, b = ctypes.byref(c), ctypes.byref(a), ctypes.byref(b)
    if op == "store":
        return lib.qwen_hip_kv8_store(c, kind, a, b, batch, n, positions, None)
    if op == "load":
        return lib.qwen_hip_kv8_load(c, kind, a, b, batch, n, flags, positions, None)
    return lib.qwen_hip_kv8_attention(c, kind, a, b, heads, batch, n, positions, max_keys, scale, ws, ws_bytes, None)


COMMON = [dict(c=cache(k=0)), dict(c=cache(v=0)), dict(c=cache(k_scale=0)), dict(c=cache(v_scale=0)),
          dict(c=cache(k=PTR + 8)), dict(c=cache(v=PTR + 1)), dict(c=cache(k_scale=PTR + 2)),
          dict(c=cache(sequences=0)), dict(c=cache(blocks=0)), dict(c=cache(blocks=(1 << 24) + 1)),
          dict(c=cache(kv_heads=0)), dict(c=cache(kv_heads=1025)), dict(c=cache(head_dim=96)), dict(c=cache(head_dim=0)),
          dict(kind=2), dict(kind=-1), dict(batch=0), dict(batch=5), dict(batch=-1), dict(n=0), dict(n=-3),
          dict(n=(1 << 24) + 1), dict(positions=None), dict(a=rows(0, token=512)), dict(b=rows(0, token=512)),
          dict(a=rows(PTR + 4, token=512)), dict(a=rows(token=513)), dict(a=rows(seq=(1 << 20) + 2, token=512)),
          dict(a=rows(token=512, head=126)), dict(a=rows(token=-512)), dict(b=rows(seq=1 << 41, token=512)),
          dict(kind=1, a=rows(token=516)), dict(c=cache(sequences=70000), batch=65536)]


@pytest.mark.parametrize("op", ["store", "load", "attend"])
@pytest.mark.parametrize("bad", COMMON)
def test_kv8_refuses(lib, op, bad):
    assert call(lib, op, **bad) == 1
    assert abi.last_error(lib)


@pytest.mark.parametrize("op,which", [("load", "a"), ("load", "b"), ("attend", "b")])
@pytest.mark.parametrize("over", [rows(token=0), rows(seq=0, token=512), rows(token=512, head=0), rows(token=128),
                                  rows(seq=1024, token=512), rows(seq=128, token=1024), rows(token=512, head=64)])
def test_kv8_refuses_overlapping_results(lib, op, which, over):
    assert call(lib, op, **{which: over}) == 1
    assert "overlap" in abi.last_error(lib)


@pytest.mark.parametrize("bad", [dict(heads=0), dict(heads=3), dict(heads=130), dict(heads=-2), dict(max_keys=0),
                                 dict(max_keys=513), dict(max_keys=-1), dict(scale=float("nan")),
                                 dict(scale=float("inf")), dict(scale=3e38), dict(n=(1 << 21) + 1),
                                 dict(c=cache(sequences=65535, kv_heads=128), batch=65535, heads=128), dict(c=cache(blocks=64), max_keys=4096, ws=None),
                                 dict(c=cache(blocks=64), max_keys=4096, ws_bytes=16),
                                 dict(c=cache(blocks=64), max_keys=4096, ws=PTR + 4)])
def test_kv8_attention_refuses(lib, bad):
    assert call(lib, "attend", **bad) == 1


def test_kv8_other_refusals(lib):
    assert call(lib, "load", flags=2) == 1
    size = ctypes.c_uint64(0)
    c = cache()
    assert lib.qwen_hip_kv8_attention_workspace(ctypes.byref(c), 0, 12, 2, 1, 512, None) == 1
    assert lib.qwen_hip_kv8_attention_workspace(ctypes.byref(c), 0, 5, 2, 1, 512, ctypes.byref(size)) == 1
    assert lib.qwen_hip_kv8_attention_workspace(ctypes.byref(c), 0, 12, 2, 1, 512, ctypes.byref(size)) == 0
    assert lib.qwen_hip_kv8_attention_workspace(None, 0, 12, 2, 1, 512, ctypes.byref(size)) == 1


def sample(lib, logits=PTR, kind=0, stride=100, n=2, vocab=100, u=PTR, ids=PTR, ws=PTR, ws_bytes=1 << 40):
    return lib.qwen_hip_sample(logits, kind, stride, n, vocab, u, None, None, None, None, ids, ws, ws_bytes, None)


@pytest.mark.parametrize("bad", [dict(logits=None), dict(u=None), dict(ids=None), dict(kind=2), dict(n=0), dict(n=-1),
                                 dict(n=65536), dict(vocab=0), dict(vocab=(1 << 24) + 1), dict(stride=-1),
                                 dict(stride=1 << 41), dict(logits=PTR + 2), dict(kind=1, logits=PTR + 1)])
def test_sample_refuses(lib, bad):
    assert sample(lib, **bad) == 1
    assert abi.last_error(lib)


def test_sample_workspace_refusals(lib):
    size = ctypes.c_uint64(0)
    assert lib.qwen_hip_sample_workspace(2, 100, None) == 1
    assert lib.qwen_hip_sample_workspace(0, 100, ctypes.byref(size)) == 1
    assert lib.qwen_hip_sample_workspace(2, 0, ctypes.byref(size)) == 1
    assert lib.qwen_hip_sample_workspace(64, 151936, ctypes.byref(size)) == 0
    if size.value:
        assert sample(lib, vocab=151936, stride=151936, ws=None) == 1
        assert sample(lib, vocab=151936, stride=151936, ws_bytes=8) == 1
