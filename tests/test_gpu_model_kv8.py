"""The device model over an 8-bit cache, and tokens drawn from its logits: one serving step as it is used.

A layer's result is checked against float64 (tests/_layer64.py) with the keys and values that the cache holds after
the call, within the FAST contract (1e-3 of the tensor's maximum); the stored rows against the float64 rows within
half a step of their block's scale beside that."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

from _kv8 import Cache
from _layer64 import Layer64
from _oracle import oracle
from work_llm_accelerator_amd.layout import HIDDEN, Q_HEADS

pytestmark = pytest.mark.gpu

TOL = 1e-3


@pytest.fixture(scope="module")
def torch():
    import torch as t

    return t


@pytest.fixture(scope="module")
def model(torch):
    from work_llm_accelerator_amd.model import DeviceModel

    m = DeviceModel(2, synthetic_seed=17)
    yield m
    m.close()


@pytest.fixture(scope="module")
def layer(torch, model):
    return Layer64.from_model(torch, model, 0)


def history(torch, batch, tokens, seed, layers=1):
    """A cache of `tokens` random tokens a sequence, with room for more."""
    from work_llm_accelerator_amd.kv8 import Kv8Cache

    cache = Kv8Cache.allocate(layers, batch, tokens + 600)
    g = torch.Generator(device="cuda").manual_seed(seed)
    if tokens:
        pos = torch.zeros(batch, dtype=torch.int32, device="cuda")
        for l in range(layers):
            k, v = (torch.randn(batch, tokens, 2, 128, generator=g, device="cuda") for _ in range(2))
            cache.store(l, k, v, pos)
    return cache


def rotated(torch, m, pos, prefill):
    """m [B, S, heads * 128] rotated at positions pos [B, S] with the mode's own cos and sin (a prefill's come from the
    reference's approximate sincos, up to 1e-3 from the true ones)."""
    o = oracle()
    row = o.oracle_prefill_rope_row if prefill else o.oracle_decode_rope_row
    row.argtypes, row.restype = [ctypes.c_int] + [np.ctypeslib.ndpointer(dtype=np.float32)] * 2, None
    table = np.zeros((*pos.shape, 2, 64), np.float32)
    for at in np.ndindex(*pos.shape):
        c, s = np.zeros(64, np.float32), np.zeros(64, np.float32)
        row(max(0, int(pos[at])), c, s)
        table[at] = c, s
    t = torch.from_numpy(table).cuda().double()
    h = m.reshape(*m.shape[:2], -1, 2, 64)
    c, s, e, d = t[:, :, None, 0], t[:, :, None, 1], h[..., 0, :], h[..., 1, :]
    return torch.cat([e * c - d * s, d * c + e * s], dim=-1)


def norm(torch, x, w, prefill):
    """RMSNorm with the mode's own square root: a prefill's is the reference's approximate one, 4% off at 1e-3 (the mean
    square of an attention output after a long random history)."""
    ms = (x * x).mean(-1) + 1e-6
    if not prefill:
        return x / ms.sqrt()[..., None] * w
    root = oracle().oracle_approx_sqrt
    root.argtypes, root.restype = [ctypes.c_float], ctypes.c_float
    r = np.array([root(float(v)) for v in ms.flatten().cpu()]).reshape(ms.shape)
    return x / torch.from_numpy(r).cuda()[..., None] * w


def check_layer(torch, layer, cache, x, got, pos, S, prefill):
    """x [B,S,1536] at positions pos[b] .. + S - 1; got: the layer's output."""
    t = torch
    B = x.shape[0]
    x = x.double()
    at = pos.long()[:, None] + t.arange(S, device="cuda")
    n = norm(t, x, layer.ln, prefill)
    at = at.cpu().numpy()
    q = rotated(t, layer._proj(n, "wq", layer.bq, terms=False)[0], at, prefill).reshape(B, S, 2, 6, 128)
    k = rotated(t, layer._proj(n, "wk", layer.bk)[0], at, prefill)
    v = layer._proj(n, "wv", layer.bv)[0].reshape(B, S, 2, 128)
    ref = Cache.of(cache)
    ctx = t.zeros(B, S, HIDDEN, dtype=t.float64, device="cuda")
    for b in range(B):
        p0 = int(pos[b])
        if p0 < 0:
            continue
        kk, vv = (t.from_numpy(ref.values(c, b)).cuda() for c in "kv")
        for c, new, held in (("k", k, kk), ("v", v, vv)):
            step = t.from_numpy(ref.scale[c][b]).cuda().repeat_interleave(64, 0)[p0:p0 + S, :, None]
            off = (held[p0:p0 + S] - new[b]).abs() - step / 2 - TOL * new[b].abs().max()
            assert float(off.max()) <= 0, f"{c} of sequence {b}"
        hidden = t.arange(p0 + S, device="cuda") > t.arange(p0, p0 + S, device="cuda")[:, None]
        heads = []
        for h in range(Q_HEADS):  # (plain products of contiguous matrices)
            sc = q[b, :, h // 6, h % 6].contiguous() @ kk[:p0 + S, h // 6].T.contiguous() / math.sqrt(128)
            heads.append(t.softmax(sc.masked_fill(hidden, -math.inf), -1) @ vv[:p0 + S, h // 6].contiguous())
        ctx[b] = t.cat(heads, dim=1)
    a = layer._proj(ctx, "wo", terms=False)[0]
    post = norm(t, a, layer.post_ln, prefill)
    gate, up = (layer._proj(post, w, terms=False)[0] for w in ("wg", "wu"))
    out = a + layer._proj(gate / (1.0 + t.exp(-gate)) * up, "wd", terms=False)[0]
    live = (pos >= 0)[:, None, None]
    off = ((got.double() - out) * live).abs().max() / (out * live).abs().max()
    assert float(off) <= TOL, float(off)


@pytest.mark.parametrize("batch,lo,hi", [(1, 0, 0), (1, 577, 577), (2, 0, 130), (24, 3, 700), (70, 10, 300), (300, 1, 90)])
def test_decode_layer(torch, model, layer, batch, lo, hi):
    from work_llm_accelerator_amd.model import FLAG_NO_BF16_ROUND

    cache = history(torch, batch, hi, 5)
    g = torch.Generator(device="cuda").manual_seed(batch)
    pos = torch.linspace(lo, hi, batch, device="cuda").to(torch.int32)
    if batch > 2:
        pos[1] = -1  # an inactive slot
    x = torch.randn(batch, HIDDEN, generator=g, device="cuda")
    before = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    hidden = x.clone()
    model.decode_kv8(hidden, pos, hi + 1, cache, flags=FLAG_NO_BF16_ROUND, layers=0)
    model.synchronize()
    check_layer(torch, layer, cache, x[:, None], hidden[:, None], pos, 1, False)
    if batch > 2:
        for was, now in zip(before, (cache.k, cache.v, cache.k_scale, cache.v_scale)):
            assert torch.equal(was[:, 1], now[:, 1])


@pytest.mark.parametrize("batch,seq,past", [(1, 1, 0), (1, 47, 0), (3, 21, 5), (1, 130, 700), (2, 257, 63), (1, 1100, 0)])
def test_prefill_layer(torch, model, layer, batch, seq, past):
    from work_llm_accelerator_amd.model import FLAG_NO_BF16_ROUND

    cache = history(torch, batch, past + (seq if seq > 500 else 0), 6)
    x = torch.randn(batch, seq, HIDDEN, generator=torch.Generator(device="cuda").manual_seed(seq), device="cuda")
    hidden = x.clone()
    model.prefill_kv8(hidden, cache, flags=FLAG_NO_BF16_ROUND, past=past, layers=0)
    model.synchronize()
    check_layer(torch, layer, cache, x, hidden, torch.full((batch,), past, dtype=torch.int32, device="cuda"), seq, True)


def test_two_layers(torch, model):
    """Both layers in one call against one call a layer: the boundary's norm is summed in another order, so codes of
    the activations differ by a step here and there."""
    x = torch.randn(2, 40, HIDDEN, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    d = torch.randn(2, HIDDEN, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    pos = torch.tensor([40, 40], dtype=torch.int32, device="cuda")
    a, b = history(torch, 2, 0, 0, layers=2), history(torch, 2, 0, 0, layers=2)
    xa, xb, da, db = x.clone(), x.clone(), d.clone(), d.clone()
    model.prefill_kv8(xa, a)
    model.decode_kv8(da, pos, 41, a)
    for l in range(2):
        model.prefill_kv8(xb, b, layers=l)
        model.decode_kv8(db, pos, 41, b, layers=l)
    model.synchronize()
    for p, q in ((xa, xb), (da, db)):
        assert float((p - q).abs().max() / q.abs().max()) <= 1e-2
    for l in range(2):
        p, q = a.load(l, pos * 0, 41), b.load(l, pos * 0, 41)
        for i in range(2):
            assert float((p[i] - q[i]).abs().max() / q[i].abs().max()) <= (0.02 if l else 0.0)


def test_sample_is_the_logits_draw(torch, model):
    """DeviceModel.sample against sample_logits of DeviceModel.logits; argmax rows against DeviceModel.greedy; more rows
    than one pass of the head takes."""
    from work_llm_accelerator_amd.model import DeviceModel
    from work_llm_accelerator_amd.sampling import sample_logits

    g = torch.Generator(device="cuda").manual_seed(3)
    small = DeviceModel(1, synthetic_seed=3)
    rng = np.random.default_rng(0)
    bits = (rng.standard_normal((640, HIDDEN)).astype(np.float32) * 0.05).view(np.uint32) >> 16
    small.set_head(bits.astype(np.uint16), np.full(HIDDEN, 0x3F80, np.uint16))
    for m, n in ((model, 1), (model, 7), (small, 20), (small, 600)):
        hidden = torch.randn(n, HIDDEN, generator=g, device="cuda")
        u = torch.rand(n, generator=g, device="cuda")
        t = torch.rand(n, generator=g, device="cuda") + 0.3
        t[::5] = 0.0
        k = torch.randint(-1, 60, (n,), generator=g, device="cuda", dtype=torch.int32)
        p, q = torch.rand(n, generator=g, device="cuda") * 0.5 + 0.5, torch.rand(n, generator=g, device="cuda") * 0.1
        ids, best = (torch.empty(n, dtype=torch.int32, device="cuda") for _ in range(2))
        logits = torch.empty(n, m.vocab, device="cuda")
        m.sample(hidden, u, ids, temperature=t, top_k=k, top_p=p, min_p=q)
        m.logits(hidden, logits)
        m.greedy(hidden, best)
        m.synchronize()
        assert torch.equal(ids, sample_logits(logits, u, t, k, p, q))
        assert torch.equal(ids[::5], best[::5])
        m.sample(hidden, u, ids)
        m.synchronize()
        assert torch.equal(ids, sample_logits(logits, u))
    small.close()


def test_generation(torch, model):
    """Prompts of different lengths, then steps of embed, decode and draw, all queued on the device: the same tokens on
    every run, those of the steps taken apart, and slots that end early left alone."""
    from work_llm_accelerator_amd.kv8 import Kv8Cache
    from work_llm_accelerator_amd.sampling import sample_logits

    g = torch.Generator(device="cuda").manual_seed(9)
    B, steps = 3, 6
    lengths = [70, 5, 33]
    prompts = [torch.randint(0, model.vocab, (n,), generator=g, device="cuda", dtype=torch.int32) for n in lengths]
    u = torch.rand(steps, B, generator=g, device="cuda")
    t, p = torch.full((B,), 0.9, device="cuda"), torch.full((B,), 0.95, device="cuda")
    k = torch.full((B,), 50, dtype=torch.int32, device="cuda")

    def generate(apart: bool):
        cache = Kv8Cache.allocate(2, B, 128)
        last = torch.empty(B, HIDDEN, device="cuda")
        for b, ids in enumerate(prompts):
            own = Kv8Cache(*(x[:, b:b + 1].contiguous() for x in (cache.k, cache.v, cache.k_scale, cache.v_scale)))
            x = torch.empty(1, len(ids), HIDDEN, device="cuda")
            model.embed(ids, x)
            model.prefill_kv8(x, own)
            model.synchronize()
            for whole, part in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), (own.k, own.v, own.k_scale, own.v_scale)):
                whole[:, b:b + 1] = part
            last[b] = x[0, -1]
        pos = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        out = []
        for i in range(steps):
            ids = torch.empty(B, dtype=torch.int32, device="cuda")
            if apart:
                logits = torch.empty(B, model.vocab, device="cuda")
                model.logits(last, logits)
                model.synchronize()
                sample_logits(logits, u[i], t, k, p, token_ids=ids)
            else:
                model.sample(last, u[i], ids, temperature=t, top_k=k, top_p=p)
            model.embed(ids, last)
            if i == 3:
                torch.cuda.synchronize()
                model.synchronize()
                pos = pos.clone()
                pos[1] = -1  # the second conversation has ended
                frozen = cache.k[:, 1].clone()
            model.decode_kv8(last, pos, 80, cache)
            model.synchronize()
            pos = torch.where(pos < 0, pos, pos + 1)
            out.append(ids)
        assert torch.equal(cache.k[:, 1], frozen)
        return torch.stack(out)

    a = generate(False)
    assert torch.equal(a[:4], generate(False)[:4]) and torch.equal(a[:, [0, 2]], generate(True)[:, [0, 2]])
    assert int(a.min()) >= 0 and int(a.max()) < model.vocab


def test_refusals(torch, model):
    from work_llm_accelerator_amd.kv8 import Kv8Cache

    cache = Kv8Cache.allocate(2, 2, 64)
    x, pos = torch.zeros(2, HIDDEN, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    for call in (lambda: model.decode_kv8(x, pos, 65, cache), lambda: model.decode_kv8(x, pos, 0, cache),
                 lambda: model.decode_kv8(torch.zeros(3, HIDDEN, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda"), 64, cache),
                 lambda: model.decode_kv8(x, pos, 64, cache, flags=0x200), lambda: model.decode_kv8(x, pos, 64, cache, layers=2),
                 lambda: model.decode_kv8(x, pos, 64, Kv8Cache.allocate(2, 2, 64, 4, 64)),
                 lambda: model.prefill_kv8(x.view(1, 2, HIDDEN), cache, past=63),
                 lambda: model.prefill_kv8(x.view(1, 2, HIDDEN), cache, past=-1),
                 lambda: model.prefill_kv8(x.view(1, 2, HIDDEN), cache, past=2 ** 32),
                 lambda: model.decode_kv8(x, pos, 2 ** 32 + 64, cache),
                 lambda: model.prefill_kv8(torch.zeros(1, 0, HIDDEN, device="cuda"), cache)):
        with pytest.raises((RuntimeError, ValueError)):
            call()
    with pytest.raises(ValueError):
        model.decode_kv8(x, pos, 64, Kv8Cache.allocate(1, 2, 64))
    with pytest.raises(ValueError):
        model.sample(x, pos, pos)
