"""Token sampling on the GPU against the definition in include/qwen_hip_sample.h, token by token in 64 bits."""

from __future__ import annotations

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as t

    return t


def drawn(x, u, t=1.0, k=0, p=1.0, q=0.0) -> int:
    """One row's token, weights as exact integers."""
    x = np.asarray(x, np.float64)
    nan = np.isnan(x)
    if nan.any():
        return int(np.argmax(nan))
    top = x.max()
    if not t > 0 or not np.isfinite(top):
        return int(np.argmax(x))
    unit = 2.0 ** min(50, 62 - math.ceil(math.log2(len(x))))
    w = np.exp((x - top) / np.float64(t))
    n = [int(v) for v in np.rint(w * unit)]
    order = np.lexsort((np.arange(len(x)), -x))
    kept = order[:k] if k > 0 else order
    if p < 1:
        goal, run, some = float(np.float64(p)) * float(sum(n[i] for i in kept)), 0, []
        for i in kept:
            if float(run) < goal or not some:
                some.append(i)
                run += n[i]
            else:
                break
        kept = some
    if q > 0:
        kept = [i for i in kept if w[i] >= min(float(q), 1.0)]
    kept = sorted(int(i) for i in kept)
    u = min(float(u), 1.0) if u > 0 else 0.0
    goal, run, token = u * float(sum(n[i] for i in kept)), 0, 0
    for i in kept:
        run += n[i]
        if n[i]:
            token = i
            if float(run) > goal:
                return i
    return token


def check(torch, x, u, dtype="float32", **params):
    rows = len(u)
    logits = torch.from_numpy(np.asarray(x, np.float32)).to(getattr(torch, dtype)).cuda()
    from work_llm_accelerator_amd.sampling import sample_logits

    dev = {n: torch.tensor(v, dtype=torch.int32 if n == "top_k" else torch.float32, device="cuda") for n, v in params.items()}
    got = sample_logits(logits, torch.tensor(u, dtype=torch.float32, device="cuda"), **dev).cpu().numpy()
    lx = logits.float().cpu().numpy()
    short = {"temperature": "t", "top_k": "k", "top_p": "p", "min_p": "q"}
    at = {n: dev[n].cpu().numpy() for n in dev}
    want = [drawn(lx[r], np.float32(u[r]), **{short[n]: at[n][r] for n in at}) for r in range(rows)]
    np.testing.assert_array_equal(got, want)
    return got


@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 65, 1000, 4097, 65537])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_settings(torch, vocab, dtype):
    rng = np.random.default_rng(vocab)
    t, k, p, q = np.meshgrid([0.5, 1.3], [0, 1, 7, 300], [1.0, 0.6], [0.0, 0.05], indexing="ij")
    rows = t.size
    x = rng.standard_normal((rows, vocab)) * 2.5
    check(torch, x, rng.random(rows), dtype, temperature=t.ravel(), top_k=k.ravel(), top_p=p.ravel(), min_p=q.ravel())


def test_defaults_are_off(torch):
    rng = np.random.default_rng(1)
    x, u = rng.standard_normal((9, 500)), rng.random(9)
    a = check(torch, x, u)
    b = check(torch, x, u, temperature=[1.0] * 9, top_k=[0] * 9, top_p=[1.0] * 9, min_p=[0.0] * 9)
    np.testing.assert_array_equal(a, b)


def test_ties(torch):
    """Few distinct logits: cuts inside groups of equal tokens keep the lowest indices."""
    rng = np.random.default_rng(2)
    x = rng.integers(-2, 3, (64, 777)).astype(np.float32)
    x[:8] = 0.25  # all equal
    x[8:12] = np.where(rng.random((4, 777)) < 0.5, 0.0, -0.0)
    u = rng.random(64)
    for k, p, q in ((0, 0.5, 0.0), (100, 1.0, 0.0), (300, 0.7, 0.0), (5, 0.9, 0.3), (0, 1.0, 0.4), (777, 0.999, 0.0), (776, 1.0, 0.0)):
        check(torch, x, u, top_k=[k] * 64, top_p=[p] * 64, min_p=[q] * 64)


def test_uniforms_at_the_ends(torch):
    x = np.tile(np.array([-np.inf, 0.0, 1.0, -np.inf, 0.5, -np.inf], np.float32), (6, 1))
    got = check(torch, x, [0.0, 1.0, np.nan, -0.5, 2.0, np.float32(1 - 2.0 ** -24)])
    assert list(got) == [1, 4, 1, 1, 4, 4]


def test_odd_parameters(torch):
    """Temperatures that take the argmax, top-k beyond the row, top-p of zero, NaN settings, min-p above 1."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((10, 300))
    u = rng.random(10)
    nan = float("nan")
    check(torch, x, u, temperature=[0.0, -1.0, nan, 1e-6, 1e6, 1.0, 1e-30, 1e30, float("inf"), -0.0])
    check(torch, x, u, top_k=[-5, 300, 301, 2 ** 31 - 1, -2 ** 31, 1, 2, 299, 0, 3])
    check(torch, x, u, top_p=[0.0, -1.0, nan, 1.0, 2.0, 1e-30, 0.5, 0.999999, 1e-6, float("inf")])
    check(torch, x, u, min_p=[0.0, -1.0, nan, 1.0, 2.0, 1e-30, 0.5, 0.999999, 1e-6, float("inf")])


def test_non_finite_logits(torch):
    rng = np.random.default_rng(4)
    x = rng.standard_normal((7, 200)).astype(np.float32)
    x[0, 50] = np.nan
    x[0, 90] = np.nan
    x[1, 20] = x[1, 10] = np.inf
    x[2] = -np.inf
    x[3, ::2] = -np.inf
    x[4] = np.nan
    x[5, :199] = -np.inf
    x[6] = -3.4e38
    x[6, 3] = 3.4e38
    for p in (1.0, 0.4):
        check(torch, x, rng.random(7), top_p=[p] * 7, top_k=[150] * 7, min_p=[0.01] * 7)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_strided_rows(torch, dtype):
    """Rows of a wider tensor at odd offsets, and one row for all draws."""
    from work_llm_accelerator_amd.sampling import sample_logits

    rng = np.random.default_rng(5)
    wide = torch.from_numpy(rng.standard_normal((5, 1001)).astype(np.float32)).to(getattr(torch, dtype)).cuda()
    u = torch.from_numpy(rng.random(5).astype(np.float32)).cuda()
    p = torch.full((5,), 0.8, device="cuda")
    part = wide[:, 3:900]
    assert torch.equal(sample_logits(part, u, top_p=p), sample_logits(part.contiguous(), u, top_p=p))
    one = wide[:1, 1:].expand(5, 1000)
    assert torch.equal(sample_logits(one, u, top_p=p), sample_logits(one.contiguous(), u, top_p=p))


def test_full_vocabulary(torch):
    """The model's vocabulary, logits rounded to bf16 as the head's are, many settings at once."""
    rng = np.random.default_rng(6)
    rows, vocab = 12, 151936
    x = rng.standard_normal((rows, vocab)) * 1.8
    x[:, rng.integers(0, vocab, 12)] = 7 + rng.standard_normal((rows, 12))
    x[3] = rng.standard_normal(vocab) * 1e-3  # nearly flat: a handful of distinct bf16 values
    check(torch, x, rng.random(rows), "bfloat16", temperature=[0.7, 1.0, 1.5] * 4, top_k=[0, 50, 1000, 100000] * 3,
          top_p=[0.95, 1.0, 0.5, 0.99, 0.9, 1.0] * 2, min_p=[0.0, 0.02] * 6)


@pytest.mark.parametrize("vocab", [524288, 524289, 1300003])
def test_longer_vocabularies(torch, vocab):
    """More tokens than segments of one width hold, aligned rows and others: no cut, cuts with and without a list, ties."""
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((5, vocab)) * 2.0
    x[2] = np.round(x[2])
    x[3] = rng.standard_normal(vocab) * 1e-5
    x[3, 5] = 9.0
    check(torch, x, rng.random(5), top_k=[0, 40, 0, 70000, 300000], top_p=[1.0, 0.9, 0.6, 0.9, 0.8], min_p=[0.0, 0.0, 0.0, 0.0, 1e-4])


def test_draws_follow_the_distribution(torch):
    """Evenly spread uniforms hit every kept token in proportion, exactly (no tolerance: the draw is an inverse)."""
    x = np.log(np.array([1.0, 2.0, 4.0, 8.0, 1.0], np.float32))
    n = 1600
    got = check(torch, np.tile(x, (n, 1)), (np.arange(n) + 0.5) / n)
    np.testing.assert_array_equal(np.bincount(got, minlength=5), [100, 200, 400, 800, 100])


def test_refusals(torch):
    from work_llm_accelerator_amd.sampling import sample_logits

    x, u = torch.zeros(4, 10, device="cuda"), torch.zeros(4, device="cuda")
    for logits, uniforms, more in ((x.half(), u, {}), (x[0], u, {}), (x.t(), u, {}), (x, u[:3], {}), (x, u.double(), {}),
                                   (x, u.cpu(), {}), (x, u, {"temperature": u[:2]}), (x, u, {"top_k": u}),
                                   (x, u, {"top_p": u.double()}), (x, u, {"min_p": x[:, 0]}), (x, u, {"token_ids": u}),
                                   (x[:, :0], u, {})):
        with pytest.raises(ValueError):
            sample_logits(logits, uniforms, **more)


def test_graph_replays(torch):
    from work_llm_accelerator_amd.sampling import sample_logits

    rng = np.random.default_rng(7)
    x, u = torch.zeros(6, 30011, device="cuda"), torch.zeros(6, device="cuda")
    p, k = torch.full((6,), 0.9, device="cuda"), torch.full((6,), 500, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        sample_logits(x, u, top_p=p, top_k=k)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ids = sample_logits(x, u, top_p=p, top_k=k)
    for _ in range(4):
        x.copy_(torch.from_numpy(rng.standard_normal((6, 30011)).astype(np.float32) * 2))
        u.copy_(torch.from_numpy(rng.random(6).astype(np.float32)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(ids, sample_logits(x, u, top_p=p, top_k=k))


def test_cuts_in_crowded_steps(torch):
    """Rows whose cut falls among thousands of logits that are equal or nearly so, rows of a few distinct values far
    apart, masks of -inf and of the lowest value, and a long flat tail without weight."""
    rng = np.random.default_rng(8)
    rows, vocab = 10, 20000
    x = np.zeros((rows, vocab), np.float32)
    x[0] = rng.standard_normal(vocab) * 1e-6
    x[0, 7] = 20.0
    x[1, ::3] = -30.0
    x[2] = np.where(rng.random(vocab) < 0.7, -np.inf, rng.standard_normal(vocab))
    x[3] = np.where(rng.random(vocab) < 0.7, np.finfo(np.float32).min, rng.standard_normal(vocab))
    x[4] = np.floor(rng.random(vocab) * 4) * 1e4
    x[5] = rng.standard_normal(vocab) - 60.0
    x[5, 3] = 0.0
    x[6] = 1e-40 * rng.integers(0, 9, vocab)
    x[7] = np.nextafter(np.float32(1), np.float32(2)) * (rng.random(vocab) < 0.5)
    x[8] = 3e38 * (2 * rng.random(vocab) - 1)
    x[9] = rng.standard_normal(vocab) * 3
    for k, p in ((0, 0.5), (15000, 1.0), (15000, 0.3), (9000, 0.999), (1, 0.5), (5000, 0.9999)):
        for t in (1.0, 0.05, 30.0):
            check(torch, x, rng.random(rows), temperature=[t] * rows, top_k=[k] * rows, top_p=[p] * rows)
