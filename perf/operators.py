"""The 8-bit K/V cache (store, load, attention over it) and token sampling, as cases that a timing program can run.

A case is one call sequence of the public Python entry points: Kv8Cache.store and .load, Kv8Cache.attend and
sample_logits.  Where `own` is false the same values come from elementary torch operations.

Sizes are those of this repository's model and benchmark (12 query heads on 2 KV heads of 128, 64 x 4096 decode,
8 x 2048 prompts, a vocabulary of 151936, 32768 positions) and of what lies around them.
"""

from __future__ import annotations

import math

import torch

own = False

BLOCK = 64  # tokens that share a scale
VOCAB = 151936
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}


# ---- the cases ------------------------------------------------------------------------------
def _cache(op: str, dtype: str, batch: int, rows: int, lo: int, hi: int, kv: int = 2, dim: int = 128, **more) -> dict:
    """`rows` new tokens of each of `batch` sequences that hold lo..hi tokens already."""
    return {**more, "op": op, "dtype": dtype, "batch": batch, "rows": rows, "lo": lo, "hi": hi, "kv": kv, "dim": dim}


def _sample(dtype: str, rows: int, vocab: int, temperature: float, top_k: int, top_p: float, min_p: float, **more) -> dict:
    return {**more, "op": "sample", "dtype": dtype, "rows": rows, "vocab": vocab, "temperature": temperature,
            "top_k": top_k, "top_p": top_p, "min_p": min_p}


def listed() -> list:
    return [
        # one conversation's new token: written, and read back with the tokens before it
        _cache("store", "f32", 1, 1, 577, 577, name="append_b1"),
        # the benchmark's decode batch, conversations of different lengths
        _cache("store", "f32", 64, 1, 100, 4095, name="append_b64"),
        # the benchmark's prompts: whole blocks
        _cache("store", "bf16", 8, 2048, 0, 0, name="append_8x2048"),
        # a prefix of odd length handed to a path that reads plain rows
        _cache("load", "bf16", 3, 777, 45, 1201, kv=4, dim=64, name="load_3x777"),
        # a long document's cache restored
        _cache("load", "f32", 4, 32768, 0, 0, name="load_4x32768"),
        # interactive generation after a 512-token prompt
        _cache("attend", "f32", 1, 1, 577, 577, group=6, name="decode_b1"),
        # the benchmark's decode: bound by the key/value stream
        _cache("attend", "f32", 64, 1, 4095, 4095, group=6, name="decode_b64_kv4096"),
        # long documents, ragged, four candidate tokens each checked in one pass
        _cache("attend", "bf16", 6, 4, 9001, 32000, group=6, name="verify_b6_long"),
        # a chunk of odd length after a history, another head layout
        _cache("attend", "f32", 2, 501, 700, 1499, kv=4, dim=64, group=7, name="chunk_2x501"),
        # a long prompt: bound by the matrix cores
        _cache("attend", "bf16", 1, 4096, 0, 0, group=6, name="prefill_1x4096"),
        # the next token of one conversation
        _sample("f32", 1, VOCAB, 0.8, 0, 0.95, 0.0, name="sample_b1"),
        # the benchmark's decode batch, every conversation with settings of its own
        _sample("f32", 64, VOCAB, 1.0, 200, 0.9, 0.02, mixed=True, name="sample_b64"),
    ]


def _log(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng) -> dict:
    kind = rng.choice(["store", "load", "decode", "decode", "few", "prompt", "prompt", "sample", "sample"])
    dtype = rng.choice(["f32", "bf16"])
    if kind == "sample":
        vocab = rng.choice([VOCAB, _log(rng, 100, VOCAB)])
        return _sample(dtype, _log(rng, 1, 64), vocab, round(rng.uniform(0.3, 1.5), 3), rng.choice([0, 1, _log(rng, 2, vocab)]),
                       round(rng.choice([1.0, rng.uniform(0.05, 0.99)]), 3), round(rng.choice([0.0, rng.uniform(0.0, 0.3)]), 3),
                       mixed=rng.random() < 0.3)
    kv, dim, group = rng.choice([1, 2, 2, 4, 8]), rng.choice([64, 128, 128]), rng.choice([1, 2, 4, 6, 6, 7, 8, 12])
    if kind in ("store", "load"):
        rows = _log(rng, 1, 16384)
        batch = _log(rng, 1, max(1, min(64, (1 << 24) // (rows * kv * dim))))
        lo = _log(rng, 1, 8000) - 1
        return _cache(kind, dtype, batch, rows, lo, lo + _log(rng, 1, 2000) - 1, kv, dim)
    if kind == "prompt":
        rows = _log(rng, 17, 4096)
        past = rng.choice([0, _log(rng, 1, 8000)])
        room = (1 << 33) // (rows * (past + rows) * kv * group * dim)
        batch = _log(rng, 1, max(1, min(8, room)))
        if room == 0:
            rows, past = rows // 8 + 1, past // 2
        return _cache("attend", dtype, batch, rows, max(0, past - past // 3), past, kv, dim, group=group)
    rows = 1 if kind == "decode" else _log(rng, 2, 16)
    hi = _log(rng, 1, 32700)
    batch = _log(rng, 1, max(1, min(200, (1 << 26) // (hi * kv * dim))))
    return _cache("attend", dtype, batch, rows, rng.randint(0, hi), hi, kv, dim, group=group)


def _held(case: dict) -> list:
    """Tokens that each sequence holds before the call: lo..hi, spread evenly."""
    n = case["batch"]
    return [case["hi"] if n == 1 else case["lo"] + (case["hi"] - case["lo"]) * b // (n - 1) for b in range(n)]


# ---- inputs ---------------------------------------------------------------------------------
def prepare(case: dict, seed: int) -> dict:
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype = TYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, generator=g, device=dev)

    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # logits as the head makes them: values rounded to bf16, a few tokens far above the rest
        logits = randn(rows, vocab) * 1.8
        tops = torch.randint(0, vocab, (rows, 12), generator=g, device=dev)
        logits.scatter_(1, tops, 7.0 + 1.2 * randn(rows, 12))
        s = {"case": case, "logits": logits.to(torch.bfloat16).to(dtype),
             "uniforms": torch.rand(rows, generator=g, device=dev)}
        row = torch.arange(rows, device=dev)
        one = torch.ones(rows, device=dev)
        mixed = bool(case.get("mixed"))
        # mixed: greedy rows, rows without top-k, without top-p, without min-p
        s["temperature"] = torch.where(row % 8 == 5, 0.0, case["temperature"] * (1.0 + 0.02 * (row % 16))) if mixed else one * case["temperature"]
        s["top_k"] = (torch.where(row % 4 == 1, 0, case["top_k"] + row % 50) if mixed else one * case["top_k"]).to(torch.int32)
        s["top_p"] = torch.where(row % 4 == 2, 1.0, case["top_p"]) * one if mixed else one * case["top_p"]
        s["min_p"] = torch.where(row % 4 == 3, 0.0, case["min_p"]) * one if mixed else one * case["min_p"]
        return s

    batch, rows, kv, dim = case["batch"], case["rows"], case["kv"], case["dim"]
    blocks = (case["hi"] + rows + BLOCK - 1) // BLOCK + 1
    # a filled cache: codes of normal values, a scale of its own for each block and head
    s = {"case": case, "blocks": blocks}
    for n in ("k", "v"):
        codes = torch.empty((batch, blocks, kv, BLOCK * dim), dtype=torch.int8, device=dev)
        for b in range(batch):
            codes[b] = (randn(blocks, kv, BLOCK * dim) * 32.0).round_().clamp_(-127, 127).to(torch.int8)
        s[n] = codes
        s[n + "_scale"] = torch.where(randn(batch, blocks, kv) < 0, 2.0 ** -5, 2.0 ** -6)
    held = torch.tensor(_held(case), dtype=torch.int32, device=dev)
    s["positions"] = held[torch.randperm(batch, generator=g, device=dev)].contiguous()
    if case["op"] == "store":
        # new rows whose sizes differ from token to token, so that some blocks' scales grow
        size = torch.exp(0.7 * randn(batch, rows, kv, 1))
        s["new_k"], s["new_v"] = ((randn(batch, rows, kv, dim) * size).to(dtype) for _ in range(2))
    if case["op"] == "attend":
        s["q"] = (randn(batch, rows, kv * case["group"], dim) * 1.5).to(dtype)
    return s


def _before(case: dict) -> int:
    """Tokens before the new ones that a store case reads back too (their codes change where a scale grows)."""
    return min(case["lo"], BLOCK)


# ---- the framework's calls ------------------------------------------------------------------
def _own(s: dict):
    from work_llm_accelerator_amd.kv8 import Kv8Cache
    from work_llm_accelerator_amd.sampling import sample_logits

    case = s["case"]
    if case["op"] == "sample":
        return sample_logits(s["logits"], s["uniforms"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                             min_p=s["min_p"])
    cache = Kv8Cache(k=s["k"][None], v=s["v"][None], k_scale=s["k_scale"][None], v_scale=s["v_scale"][None])
    if case["op"] == "attend":
        return cache.attend(0, s["q"], s["positions"], max_keys=case["hi"] + case["rows"])
    if case["op"] == "store":
        cache.store(0, s["new_k"], s["new_v"], s["positions"])
        n = _before(case)
        return cache.load(0, s["positions"] - n, n + case["rows"], dtype=TYPES[case["dtype"]])
    return cache.load(0, s["positions"], case["rows"], dtype=TYPES[case["dtype"]])


# ---- the plain forms ------------------------------------------------------------------------
def _codes(s: dict, n: str, blocks: int):
    """[batch, blocks, 64 tokens, kv, dim] view of the first `blocks` blocks' codes.  K: halves of 64 dimensions, token
    by token; V: dimension by dimension, token 16t+4g+i at place 16g+4t+i."""
    c = s[n][:, :blocks]
    b, nb, kv = c.shape[:3]
    if n == "k":
        return c.view(b, nb, kv, -1, 64, 64).permute(0, 1, 4, 2, 3, 5)  # b, nb, token, kv, half, 64
    return c.view(b, nb, kv, -1, 4, 4, 4).permute(0, 1, 5, 4, 6, 2, 3)  # b, nb, t, g, i, kv, dim


def _values(s: dict, n: str, blocks: int):
    """[batch, blocks * 64, kv, dim] values of the first `blocks` blocks in fp32."""
    c = _codes(s, n, blocks)
    kv, dim = s["case"]["kv"], s["case"]["dim"]
    v = c.reshape(c.shape[0], blocks, BLOCK, kv, dim).float() * s[n + "_scale"][:, :blocks, None, :, None]
    return v.reshape(c.shape[0], blocks * BLOCK, kv, dim)


def _read(s: dict, first, rows: int, dtype):
    """Rows first..first+rows-1 of every sequence."""
    at = first.long()[:, None] + torch.arange(rows, device=first.device)
    b = torch.arange(at.shape[0], device=first.device)[:, None]
    return tuple(_values(s, n, s["blocks"])[b, at].to(dtype) for n in ("k", "v"))


def _plain_store(s: dict, n: str, new) -> None:
    """Writes `new` [batch, rows, kv, dim] behind the tokens held, in codes: the blocks that it touches, whole."""
    case, pos = s["case"], s["positions"].long()
    rows, kv, dim, batch = case["rows"], case["kv"], case["dim"], pos.numel()
    touched = (rows + BLOCK - 2) // BLOCK + 1  # at most, whatever the position in its block
    first = pos // BLOCK
    block = first[:, None] + torch.arange(touched, device=pos.device)  # prepare() leaves a block behind the last one
    b = torch.arange(batch, device=pos.device)[:, None]
    token = (first[:, None] * BLOCK + torch.arange(touched * BLOCK, device=pos.device)).view(batch, touched, BLOCK)
    src = token - pos[:, None, None]
    is_new = (src >= 0) & (src < rows)
    x = torch.where(is_new[..., None, None], new.float()[b[..., None], src.clamp(0, rows - 1)], 0.0)
    # the least power of two s with max|x| <= 127 s: max = m 2^e, 1/2 <= m < 1, 127 = (127/128) 2^7
    m, e = torch.frexp(x.abs().amax(dim=(2, 4)))
    e = torch.where(m > 127 / 128, e - 6, e - 7).clamp(min=-126)
    need = torch.where(m == 0, 2.0 ** -126, ((e + 127) << 23).to(torch.int32).view(torch.float32))
    old = s[n + "_scale"][b, block]
    fresh = (token[..., 0] >= pos[:, None])[..., None]
    some = is_new.any(2)[..., None]
    scale = torch.where(some, torch.where(fresh, need, torch.maximum(need, old)), old)
    was = _codes(s, n, s["blocks"]).reshape(batch, s["blocks"], BLOCK, kv, dim)[b, block].float()
    held = torch.where((token < pos[:, None, None])[..., None, None], torch.round(was * (old / scale)[:, :, None, :, None]), was)
    code = torch.where(is_new[..., None, None], torch.round(x / scale[:, :, None, :, None]), held).to(torch.int8)
    # back into the layout; a block that no new token touches keeps what it holds
    if n == "k":
        flat = code.reshape(batch, touched, BLOCK, kv, dim // 64, 64).permute(0, 1, 3, 4, 2, 5)
    else:
        flat = code.reshape(batch, touched, 4, 4, 4, kv, dim).permute(0, 1, 5, 6, 3, 2, 4)
    s[n][b, block] = flat.reshape(batch, touched, kv, BLOCK * dim)
    s[n + "_scale"][b, block] = scale


def _plain_attend(s: dict):
    case, q, pos = s["case"], s["q"], s["positions"].long()
    batch, rows, kv, dim, group = case["batch"], case["rows"], case["kv"], case["dim"], case["group"]
    blocks = (case["hi"] + rows + BLOCK - 1) // BLOCK
    k, v = (_values(s, n, blocks).permute(0, 2, 1, 3).contiguous() for n in ("k", "v"))  # [batch, kv, keys, dim]
    qf = q.float().view(batch, rows, kv, group, dim).permute(0, 2, 1, 3, 4).reshape(batch, kv, rows * group, dim)
    p = torch.matmul(qf, k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(dim))
    last = pos[:, None] + torch.arange(rows, device=pos.device)
    dead = torch.arange(blocks * BLOCK, device=pos.device) > last[..., None]
    p.masked_fill_(dead[:, None].repeat_interleave(group, dim=2), -math.inf)
    p = torch.exp(p - p.amax(dim=3, keepdim=True))
    o = torch.matmul(p / p.sum(dim=3, keepdim=True), v)
    return o.view(batch, kv, rows, group, dim).permute(0, 2, 1, 3, 4).reshape(batch, rows, kv * group, dim).to(q.dtype)


def _plain_sample(s: dict):
    # sums of up to 151936 weights decide next to a border: 64 bits
    value, index = torch.sort(s["logits"].float(), dim=1, descending=True, stable=True)
    t = s["temperature"].double()[:, None]
    greedy = t <= 0
    w = torch.exp((value.double() - value[:, :1].double()) / torch.where(greedy, 1.0, t))
    place = torch.arange(w.shape[1], device=w.device)
    k = s["top_k"][:, None]
    kept = torch.where((place < k) | (k <= 0), w, 0.0)
    before = torch.cumsum(kept, dim=1) - kept
    p = s["top_p"].double()[:, None]
    kept = torch.where((before < p * kept.sum(dim=1, keepdim=True)) | (p >= 1) | (place == 0), kept, 0.0)
    kept = torch.where((w >= s["min_p"].double()[:, None]) & (~greedy | (place == 0)), kept, 0.0)
    run = torch.cumsum(torch.zeros_like(w).scatter(1, index, kept), dim=1)
    goal = s["uniforms"].double()[:, None] * run[:, -1:]
    return (run <= goal).sum(dim=1).to(torch.int32)


def run(state: dict):
    if own:
        return _own(state)
    case = state["case"]
    if case["op"] == "sample":
        return _plain_sample(state)
    if case["op"] == "attend":
        return _plain_attend(state)
    if case["op"] == "store":
        for n in ("k", "v"):
            _plain_store(state, n, state["new_" + n])
        n = _before(case)
        return _read(state, state["positions"] - n, n + case["rows"], TYPES[case["dtype"]])
    return _read(state, state["positions"], case["rows"], TYPES[case["dtype"]])


# ---- what a pass cannot do without ----------------------------------------------------------
def work(case: dict) -> dict:
    size = SIZE[case["dtype"]]
    if case["op"] == "sample":
        return {"bytes": case["rows"] * (case["vocab"] * size + 24), "flops": 3 * case["rows"] * case["vocab"]}
    batch, rows, width = case["batch"], case["rows"], case["kv"] * case["dim"]
    if case["op"] == "load":
        n = 2 * batch * rows * width
        return {"bytes": n * (1 + size), "flops": n}
    if case["op"] == "store":  # rows in, codes out; those and the ones before them read, and written as rows
        n, more = 2 * batch * rows * width, 2 * batch * _before(case) * width
        return {"bytes": n * (size + 1) + (n + more) * (1 + size), "flops": 3 * n}
    held = _held(case)
    keys = sum(h + rows for h in held)
    pairs = sum(rows * h + rows * (rows + 1) // 2 for h in held)
    heads = case["kv"] * case["group"]
    return {"bytes": 2 * keys * (width + case["kv"] * 4 / BLOCK) + 2 * batch * rows * heads * case["dim"] * size,
            "flops": 4 * pairs * heads * case["dim"]}


# ---- the definitions in 64 bits -------------------------------------------------------------
def _exact_rows(s: dict, n: str, b: int):
    """[blocks, 64, kv, dim] codes of sequence b, each found at its place by formula."""
    kv, dim = s["case"]["kv"], s["case"]["dim"]
    dev = s[n].device
    t, d = torch.arange(64, device=dev)[:, None], torch.arange(dim, device=dev)
    at = (d // 64 * 64 + t) * 64 + d % 64 if n == "k" else d * 64 + 16 * (t // 4 % 4) + 4 * (t // 16) + t % 4
    return s[n][b][:, :, at].permute(0, 2, 1, 3).double()  # [blocks, kv, 64, dim] -> tokens before heads


def exact(case: dict, seed: int):
    if case["op"] == "sample":
        return None
    s = prepare(case, seed)
    rows, out = case["rows"], []
    for b in range(case["batch"]):
        pos = int(s["positions"][b])
        code, scale = {n: _exact_rows(s, n, b) for n in "kv"}, {n: s[n + "_scale"][b].double() for n in "kv"}
        if case["op"] == "store":
            for n in "kv":
                new = s["new_" + n][b].double()
                for j in range(pos // 64, (pos + rows - 1) // 64 + 1):
                    lo, hi = max(pos, 64 * j), min(pos + rows, 64 * j + 64)
                    x = new[lo - pos:hi - pos]
                    most = x.abs().amax(dim=(0, 2)).clamp(min=127 * 2.0 ** -126)
                    need = torch.full_like(most, 2.0 ** -126)
                    for step in (128, 64, 32, 16, 8, 4, 2, 1):  # the least exponent, by halving
                        less = need * 2.0 ** (step - 1)  # too small by a factor of two or more: go up
                        need = torch.where(most > 127 * less, less * 2, need)
                    to = need if lo == 64 * j else torch.maximum(need, scale[n][j])
                    code[n][j] = torch.round(code[n][j] * (scale[n][j] / to)[:, None])
                    code[n][j, lo - 64 * j:hi - 64 * j] = torch.round(x / to[:, None])
                    scale[n][j] = to
        value = {n: (code[n] * scale[n][:, None, :, None]).flatten(0, 1) for n in "kv"}
        if case["op"] != "attend":
            first = pos - (_before(case) if case["op"] == "store" else 0)
            out.append([value[n][first:pos + rows].clone() for n in "kv"])
            continue
        group, dim = case["group"], case["dim"]
        heads = []
        for h in range(case["kv"] * group):
            k, v = value["k"][:pos + rows, h // group], value["v"][:pos + rows, h // group]
            z = s["q"][b, :, h].double() @ k.T / math.sqrt(dim)
            z += torch.full_like(z, -math.inf).triu(pos + 1)
            heads.append(torch.softmax(z, dim=1) @ v)
        out.append(torch.stack(heads, dim=1))
    if case["op"] == "attend":
        return torch.stack(out)
    return tuple(torch.stack([o[i] for o in out]) for i in range(2))
