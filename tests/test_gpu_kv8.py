"""The 8-bit K/V cache on the GPU: codes and scales bit for bit, what the calls leave alone, and the attention
against 64-bit arithmetic (tests/_kv8.py) with tolerances from the operands' rounding."""

from __future__ import annotations

import math

import numpy as np
import pytest

from _kv8 import Cache, tolerance

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as t

    return t


def filled(torch, sequences, blocks, kv, dim, seed, layers=1):
    """A cache with random codes in every byte and a random scale for each block."""
    from work_llm_accelerator_amd.kv8 import Kv8Cache

    rng = np.random.default_rng(seed)
    shape = (layers, sequences, blocks, kv)
    code = [torch.from_numpy(rng.integers(-127, 128, (*shape, 64 * dim), dtype=np.int8)).cuda() for _ in range(2)]
    scale = [torch.from_numpy(2.0 ** rng.integers(-9, -3, shape).astype(np.float32)).cuda() for _ in range(2)]
    return Kv8Cache(*code, *scale)


def rows_of(torch, rng, shape, dtype, spread=1.0):
    """Rows in `dtype`, token sizes spread over powers of ten, and the same values in float32 numpy."""
    x = rng.standard_normal(shape) * 10.0 ** (spread * rng.uniform(-1, 1, (*shape[:2], shape[2], 1)))
    t = torch.from_numpy(x.astype(np.float32)).to(getattr(torch, dtype)).cuda()
    return t, t.float().cpu().numpy()


def ints(torch, values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def same(cache, ref, layer=0):
    got = Cache.of(cache, layer)
    for n in "kv":
        np.testing.assert_array_equal(got.scale[n], ref.scale[n], err_msg=n + " scales")
        np.testing.assert_array_equal(got.code[n], ref.code[n], err_msg=n + " codes")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("kv,dim", [(2, 128), (1, 64), (3, 64), (5, 128)])
@pytest.mark.parametrize("rows", [1, 2, 63, 64, 65, 200])
def test_store(torch, dtype, kv, dim, rows):
    positions = [0, 1, 63, 64, 100, 190, 255, -1, 256, 2 ** 31 - 1]  # the cache ends at 256
    cache = filled(torch, len(positions), 4, kv, dim, rows * 10 + kv)
    ref = Cache.of(cache)
    rng = np.random.default_rng(rows)
    k, kn = rows_of(torch, rng, (len(positions), rows, kv, dim), dtype)
    v, vn = rows_of(torch, rng, (len(positions), rows, kv, dim), dtype)
    cache.store(0, k, v, ints(torch, positions))
    ref.store(kn, vn, positions)
    same(cache, ref)  # every byte: what lies behind the new tokens too


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_store_edges_of_the_code(torch, dtype):
    """Zeros, denormals, the largest values, ties between codes, and magnitudes next to 127 steps."""
    cache = filled(torch, 7, 1, 1, 64, 3)
    ref = Cache.of(cache)
    x = np.zeros((7, 3, 1, 64), np.float32)
    x[1] = 1e-40
    x[2, 1] = 3.0e38
    x[3, 0, 0, :4] = [127.0, 0.5, 1.5, -2.5]
    x[4, 0, 0, :3] = [127.5, 1.0, -3.0]
    x[5, 2, 0, :2] = [-2.0 ** -126, 2.0 ** -127]
    x[6, :, 0, :] = -0.0
    t = torch.from_numpy(x).to(getattr(torch, dtype)).cuda()
    pos = [0, 0, 5, 0, 0, 0, 9]
    cache.store(0, t, -t, ints(torch, pos))
    ref.store(t.float().cpu().numpy(), -t.float().cpu().numpy(), pos)
    same(cache, ref)


def test_store_growth_stays_within_a_step(torch):
    """64 tokens stored one by one, each larger than the last: every value within one step of what was stored."""
    from work_llm_accelerator_amd.kv8 import Kv8Cache

    rng = np.random.default_rng(8)
    cache = Kv8Cache.allocate(1, 1, 64, 2, 64)
    ref = Cache.of(cache)
    x = (rng.standard_normal((1, 64, 2, 64)) * 1.2 ** np.arange(64)[None, :, None, None]).astype(np.float32)
    t = torch.from_numpy(x).cuda()
    for i in range(64):
        cache.store(0, t[:, i:i + 1], -t[:, i:i + 1], ints(torch, [i]))
        ref.store(x[:, i:i + 1], -x[:, i:i + 1], [i])
    same(cache, ref)
    k, v = cache.load(0, ints(torch, [0]), 64)
    step = ref.scale["k"][0, 0][None, :, None]
    assert np.all(np.abs(k[0].cpu().numpy() - x[0]) <= step)
    assert np.all(np.abs(v[0].cpu().numpy() + x[0]) <= step)


def test_store_in_one_call_or_by_token(torch):
    """Whole blocks in one call have the scale of their largest value; a block restarted forgets the old one."""
    rng = np.random.default_rng(9)
    cache = filled(torch, 2, 3, 2, 128, 4)
    x, xn = rows_of(torch, rng, (2, 150, 2, 128), "float32")
    cache.store(0, x, x, ints(torch, [0, 0]))
    small = x * 1e-3
    cache.store(0, small, small, ints(torch, [0, 64]))
    ref = Cache.of(filled(torch, 2, 3, 2, 128, 4))
    ref.store(xn, xn, [0, 0])
    ref.store(small.cpu().numpy(), small.cpu().numpy(), [0, 64])
    same(cache, ref)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_non_finite_values_stay_visible(torch, value):
    cache = filled(torch, 2, 2, 2, 128, 5)
    rng = np.random.default_rng(1)
    x, xn = rows_of(torch, rng, (2, 3, 2, 128), "float32", 0.0)
    x[0, 1, 1, 17] = value
    ref = Cache.of(cache)
    cache.store(0, x, x.abs(), ints(torch, [60, 60]))  # tokens 60..62 of block 0
    ref.store(x.cpu().numpy(), x.abs().cpu().numpy(), [60, 60])
    same(cache, ref)
    k, _ = cache.load(0, ints(torch, [0, 0]), 63)
    assert torch.isnan(k[0, :, 1]).all() and torch.isfinite(k[0, :, 0]).all() and torch.isfinite(k[1]).all()
    # further tokens of the block, a NaN scale before them
    y, yn = rows_of(torch, rng, (2, 1, 2, 128), "float32", 0.0)
    cache.store(0, y, y, ints(torch, [63, 63]))
    ref.store(yn, yn, [63, 63])
    same(cache, ref)
    out = cache.attend(0, torch.ones(2, 2, 2, 128, device="cuda"), ints(torch, [59, 59]), 64)
    assert torch.isnan(out[0, :, 1]).all() and torch.isfinite(out[0, :, 0]).all() and torch.isfinite(out[1]).all()
    # stored anew from the block's first token: finite again
    cache.store(0, y, y, ints(torch, [0, 0]))
    ref.store(yn, yn, [0, 0])
    same(cache, ref)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("kv,dim", [(2, 128), (3, 64)])
@pytest.mark.parametrize("rows", [1, 64, 65, 150])
def test_load(torch, dtype, kv, dim, rows):
    positions = [0, 1, 63, 100, 127, -1, -70, -300, 500, -2 ** 31, 2 ** 31 - 1]
    cache = filled(torch, len(positions), 3, kv, dim, 11)
    ref = Cache.of(cache)
    d = getattr(torch, dtype)
    want = np.zeros((2, len(positions), rows, kv, dim))
    for b, pos in enumerate(positions):
        for i in range(rows):
            if 0 <= pos + i < ref.tokens:
                want[0, b, i], want[1, b, i] = ref.values("k", b)[pos + i], ref.values("v", b)[pos + i]
            else:
                want[:, b, i] = 7.0  # left alone
    k, v = (torch.full((len(positions), rows, kv, dim), 7.0, dtype=d, device="cuda") for _ in range(2))
    cache.load(0, ints(torch, positions), k=k, v=v)
    np.testing.assert_array_equal(k.double().cpu().numpy(), want[0])  # exact in bf16 too
    np.testing.assert_array_equal(v.double().cpu().numpy(), want[1])
    k, v = cache.load(0, ints(torch, positions), rows, dtype=d)
    want[want == 7.0] = 0.0
    np.testing.assert_array_equal(np.where(k.double().cpu().numpy() == 7.0, 0.0, k.double().cpu().numpy()), want[0])
    np.testing.assert_array_equal(np.where(v.double().cpu().numpy() == 7.0, 0.0, v.double().cpu().numpy()), want[1])


def test_strided_rows(torch):
    """Slices of a fused projection, heads before tokens, broadcast rows, single tokens of a longer tensor."""
    rng = np.random.default_rng(21)
    B, S, H, D = 2, 70, 2, 128
    for layout in ("fused", "heads_first", "broadcast", "one_token"):
        cache = filled(torch, B, 3, H, D, 6)
        ref = Cache.of(cache)
        if layout == "fused":
            qkv = torch.from_numpy(rng.standard_normal((B, S, 6 * D + 2 * H * D)).astype(np.float32)).cuda()
            k, v = (qkv[..., 6 * D + i * H * D:6 * D + (i + 1) * H * D].view(B, S, H, D) for i in range(2))
        elif layout == "heads_first":
            k, v = (torch.from_numpy(rng.standard_normal((B, H, S, D)).astype(np.float32)).cuda().transpose(1, 2) for _ in range(2))
        elif layout == "broadcast":
            k = torch.from_numpy(rng.standard_normal((1, S, 1, D)).astype(np.float32)).cuda().expand(B, S, H, D)
            v = torch.from_numpy(rng.standard_normal((B, 1, H, D)).astype(np.float32)).cuda().expand(B, S, H, D)
        else:
            t = torch.from_numpy(rng.standard_normal((B, S, H, D)).astype(np.float32)).cuda()
            k, v = t[:, 5:6], t[:, 9:10]
        cache.store(0, k, v, ints(torch, [3, 100]))
        ref.store(k.cpu().numpy(), v.cpu().numpy(), [3, 100])
        same(cache, ref)
        out = torch.full((B, H, S, D), 5.0, device="cuda")  # read back into heads-first rows
        n = k.shape[1]
        cache.load(0, ints(torch, [3, 100]), k=out[:, :, :n].transpose(1, 2), v=torch.empty(B, n, H, D, device="cuda"))
        for b, pos in enumerate((3, 100)):
            np.testing.assert_array_equal(out[b, :, :n].cpu().numpy(), ref.values("k", b)[pos:pos + n].transpose(1, 0, 2))
        assert (out[:, :, n:] == 5.0).all()


def check_attend(torch, cache, q, positions, max_keys, layer=0, scale=None, **more):
    dtype = "f32" if q.dtype == torch.float32 else "bf16"
    s = 1.0 / math.sqrt(cache.head_dim) if scale is None else scale
    want, slack, floor, reach = Cache.of(cache, layer).attend(q.float().cpu().numpy(), positions, s)
    got = cache.attend(layer, q, ints(torch, positions), max_keys, scale=scale, **more).float().cpu().numpy()
    tol = tolerance(dtype, cache.head_dim, slack, floor, reach, want)
    off = np.abs(got - want) - tol
    worst = np.unravel_index(np.argmax(off), off.shape)
    assert off[worst] <= 0, f"{worst}: {got[worst]} against {want[worst]}, tolerance {tol[worst]}"
    return got


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("kv,group,dim", [(2, 6, 128), (1, 1, 64), (2, 7, 64), (3, 12, 128), (1, 64, 64)])
@pytest.mark.parametrize("rows", [1, 2, 5, 33])
def test_attend(torch, dtype, kv, group, dim, rows):
    positions = [0, 1, 62, 63, 64, -1, 200, 319 - rows]
    cache = filled(torch, len(positions), 5, kv, dim, group + rows)
    rng = np.random.default_rng(rows)
    q, _ = rows_of(torch, rng, (len(positions), rows, kv * group, dim), dtype, 0.3)
    got = check_attend(torch, cache, q, positions, 320)
    assert not got[5].any()  # inactive: zeros


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,keys", [(1, 4000), (4, 2500), (1, 9000), (130, 1000), (257, 700), (64, 64), (300, 300)])
def test_attend_long(torch, dtype, rows, keys):
    """Key splits and their merge; prompts from position 0 and after a history."""
    blocks = (keys + 63) // 64
    cache = filled(torch, 2, blocks, 2, 128, keys)
    rng = np.random.default_rng(keys)
    q, _ = rows_of(torch, rng, (2, rows, 4, 128), dtype, 0.3)
    check_attend(torch, cache, q, [keys - rows, max(0, keys // 3 - rows)], keys)


def test_attend_peaked_and_flat(torch):
    """Scores far apart (one token takes all), all equal, and a scale of zero or below."""
    cache = filled(torch, 1, 20, 1, 128, 2)
    rng = np.random.default_rng(2)
    q, _ = rows_of(torch, rng, (1, 3, 2, 128), "float32", 0.0)
    check_attend(torch, cache, q * 300.0, [1200], 1280)
    check_attend(torch, cache, q * 0.0, [1200], 1280)
    check_attend(torch, cache, q, [1200], 1280, scale=0.0)
    check_attend(torch, cache, q, [1200], 1280, scale=-0.3)
    check_attend(torch, cache, q * 1e-38, [1200], 1280, scale=1e30)
    check_attend(torch, cache, q * 1e30, [1200], 1280, scale=1e-30)


def test_attend_scales_far_apart(torch):
    """Block scales from 2^-40 to 2^30: the products carry them, not the fp16 operands."""
    cache = filled(torch, 1, 6, 2, 64, 12)
    e = torch.tensor([-40, 5, -3, 0, 12, -20], dtype=torch.float32, device="cuda")
    cache.v_scale[0, 0] = torch.exp2(e)[:, None]
    cache.k_scale[0, 0] = 2.0 ** -9
    rng = np.random.default_rng(3)
    for dtype in ("float32", "bfloat16"):
        q, _ = rows_of(torch, rng, (1, 40, 6, 64), dtype, 0.0)
        check_attend(torch, cache, q, [340], 384)


def test_attend_ignores_what_lies_behind(torch):
    """Bytes and NaN scales behind a sequence's tokens, other sequences, and tokens at or behind max_keys."""
    cache = filled(torch, 2, 4, 2, 128, 13)
    rng = np.random.default_rng(4)
    q, _ = rows_of(torch, rng, (2, 3, 12, 128), "float32", 0.0)
    want = check_attend(torch, cache, q, [60, 125], 256)
    for n in (cache.k_scale, cache.v_scale):
        n[0, 0, 1:] = float("nan")
        n[0, 1, 2:] = float("nan")
    got = cache.attend(0, q, ints(torch, [60, 125]), 256).cpu().numpy()
    # sequence 0: tokens 60..62, block 0 only; sequence 1: 125, 126, 127, blocks 0 and 1
    np.testing.assert_array_equal(got, want)
    cache.v_scale[0, 1, 1:] = float("nan")  # block 1 of sequence 1 is attended by all three rows: all NaN
    assert np.isnan(cache.attend(0, q, ints(torch, [60, 125]), 256).cpu().numpy()[1]).all()
    # rows that do not reach a NaN block, beside rows that do
    got = cache.attend(0, q, ints(torch, [60, 62]), 256).cpu().numpy()
    assert np.isfinite(got[1, :2]).all() and np.isnan(got[1, 2]).all()
    # max_keys cuts
    cut = cache.attend(0, q, ints(torch, [60, 125]), 64).cpu().numpy()
    assert np.isfinite(cut).all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("sequences,blocks,dim", [(15, 25, 64), (15, 25, 128), (80, 25, 64), (80, 25, 128), (40, 80, 64)])
def test_attend_large_tiles(torch, dtype, sequences, blocks, dim):
    """Tiles of many rows, split over the keys or not, with one key group a workgroup (15 sequences) or several: ragged
    lengths, V scales far apart, NaN scales behind a sequence and in the reach of its last rows only."""
    rows, rng = 17, np.random.default_rng(blocks + dim)
    cache = filled(torch, sequences, blocks, 2, dim, sequences + blocks)
    cache.v_scale[0] *= torch.exp2(torch.from_numpy(rng.choice([0.0, 0.0, -1.0, -7.0, 9.0, -30.0], (sequences, blocks, 2))).float()).cuda()
    end = 64 * blocks - rows
    positions = [[-1, 0, 1, 47, 48, 63, 64, 600, 1000, end - 64, end - 1, end][b % 12] for b in range(sequences)]
    for b, pos in enumerate(positions):
        last = (pos + rows - 1) // 64  # block of the last row
        if b % 2 and pos >= 0:
            cache.k_scale[0, b, last + 1:] = float("nan")
            cache.v_scale[0, b, last + 1:] = float("nan")
        elif b % 4 == 0 and pos // 64 < last:
            (cache.k_scale if b % 8 else cache.v_scale)[0, b, last] = float("nan")
    q, qn = rows_of(torch, rng, (sequences, rows, 4, dim), dtype, 0.3)
    want, slack, floor, reach = Cache.of(cache).attend(qn, positions, 0.1)
    got = cache.attend(0, q, ints(torch, positions), 64 * blocks, scale=0.1).float().cpu().numpy()
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    assert np.isnan(want).any() and not np.isnan(want).all(axis=(1, 2, 3)).any()
    tol = tolerance("f32" if dtype == "float32" else "bf16", dim, slack, floor, reach, want)
    assert (np.abs(got - want) <= tol)[~np.isnan(want)].all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("sequences,blocks,rows", [(2, 6, 3), (2, 6, 40), (80, 25, 17)])
def test_attend_blocks_of_zeros(torch, dtype, sequences, blocks, rows):
    """Blocks whose values are all zero, stored (the least scale) or never stored (a scale of 0), first, last and between
    others: they weigh in the sum of the probabilities like any other."""
    cache = filled(torch, sequences, blocks, 2, 64, 40 + rows)
    for b in range(sequences):
        for j in range(b % 4, blocks, 4 if b % 3 else 1 + b % 5):
            cache.v[0, b, j] = 0
            cache.v_scale[0, b, j] = 0.0 if b % 2 else 2.0 ** -126
    cache.k[0, 1, 1], cache.k_scale[0, 1, 1] = 0, 2.0 ** -126
    cache.k[0, 1, 2], cache.k_scale[0, 1, 2] = 0, 0.0
    q, _ = rows_of(torch, np.random.default_rng(rows), (sequences, rows, 4, 64), dtype, 0.0)
    check_attend(torch, cache, q, [64 * blocks - rows - 11 * (b % 5) for b in range(sequences)], 64 * blocks)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,sequences,blocks", [(40, 1, 20), (17, 80, 25)])
def test_attend_large_tiles_peaked_and_flat(torch, dtype, rows, sequences, blocks):
    """Tiles of many rows: one token takes all, all tokens equal, scales of the attention of zero and below, maxima that
    rise from block to block while the V scales fall and the other way round."""
    cache = filled(torch, sequences, blocks, 2, 64, 7 + rows)
    q, _ = rows_of(torch, np.random.default_rng(rows), (sequences, rows, 4, 64), dtype, 0.0)
    pos = [64 * blocks - rows - 3 * (b % 9) for b in range(sequences)]
    few = slice(0, min(3, sequences))

    def check(x, scale):
        part = type(cache)(*(t[:, few].contiguous() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)))
        want, slack, floor, reach = Cache.of(part).attend(x[few].float().cpu().numpy(), pos[few], scale)
        got = cache.attend(0, x, ints(torch, pos), 64 * blocks, scale=scale)[few].float().cpu().numpy()
        tol = tolerance("f32" if dtype == "float32" else "bf16", 64, slack, floor, reach, want)
        assert (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) - tol)

    for x, scale in ((q * 300, 0.125), (q * 0, 0.125), (q, 0.0), (q, -0.3)):
        check(x, scale)
    step = torch.arange(blocks, dtype=torch.float32, device="cuda")
    for sign in (1, -1):
        cache.k_scale[0] = torch.exp2(-9 + step * (6 / blocks))[:, None].log2().round().exp2()
        cache.v_scale[0] = torch.exp2(sign * 4 * (step - blocks // 2))[:, None]
        check(q * 8, 0.125)


def test_attend_non_finite_queries(torch):
    cache = filled(torch, 1, 2, 1, 64, 14)
    q = torch.ones(1, 4, 1, 64, device="cuda")
    q[0, 1, 0, 3] = float("nan")
    q[0, 2, 0, 5] = float("inf")
    got = cache.attend(0, q, ints(torch, [70]), 128).cpu().numpy()
    assert np.isfinite(got[0, [0, 3]]).all() and np.isnan(got[0, [1, 2]]).all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_attend_strided_and_in_place(torch, dtype):
    cache = filled(torch, 2, 3, 2, 64, 15, layers=2)
    rng = np.random.default_rng(5)
    flat, _ = rows_of(torch, rng, (2, 9, 16, 64), dtype, 0.0)
    q = flat[:, 1:6, 2:14]
    want = cache.attend(1, q, ints(torch, [100, 20]), 192)
    hf = torch.zeros(2, 12, 5, 64, dtype=q.dtype, device="cuda")
    cache.attend(1, q, ints(torch, [100, 20]), 192, out=hf.transpose(1, 2))
    assert torch.equal(hf.transpose(1, 2), want)
    before = flat.clone()
    cache.attend(1, q, ints(torch, [100, 20]), 192, out=q)
    assert torch.equal(q, want)
    before[:, 1:6, 2:14] = want
    assert torch.equal(flat, before)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("sequences,blocks,rows", [(4, 20, 40), (80, 25, 17), (3, 5, 300)])
def test_attend_large_tiles_in_place_and_captured(torch, dtype, sequences, blocks, rows):
    """Results over the queries themselves, with and without key splits (also where one split holds all of a short
    sequence), in a captured call that is replayed at other lengths."""
    cache = filled(torch, sequences, blocks, 2, 64, 3 + rows)
    rng = np.random.default_rng(rows)
    source, _ = rows_of(torch, rng, (sequences, rows, 6, 64), dtype, 0.0)
    q, pos = source.clone(), ints(torch, [0] * sequences)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.attend(0, q, pos, 64 * blocks, out=q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        cache.attend(0, q, pos, 64 * blocks, out=q)
    for turn in range(3):
        pos.copy_(ints(torch, rng.integers(-1, 64 * blocks - rows + 1, sequences).tolist()))
        q.copy_(source)
        want = cache.attend(0, source, pos, 64 * blocks)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(q, want)


def test_python_refusals(torch):
    from work_llm_accelerator_amd.kv8 import Kv8Cache

    cache = Kv8Cache.allocate(1, 2, 100, 2, 128)
    assert cache.positions == 128
    x, pos = torch.zeros(2, 3, 2, 128, device="cuda"), ints(torch, [0, 0])
    for bad in (x[:, :, :1], x[..., :64], x.half(), x.cpu(), x.transpose(2, 3), x[0]):
        with pytest.raises(ValueError):
            cache.store(0, bad, bad, pos)
    for bad in (pos.long(), pos[:1], pos.cpu(), torch.zeros(4, dtype=torch.int32, device="cuda")[::2]):
        with pytest.raises(ValueError):
            cache.store(0, x, x, bad)
    with pytest.raises(ValueError):
        cache.store(1, x, x, pos)
    with pytest.raises(ValueError):
        cache.store(0, x, x.bfloat16(), pos)
    with pytest.raises(ValueError):
        cache.attend(0, x, pos, 129)
    with pytest.raises(ValueError):
        cache.attend(0, x, pos, 64, out=x.bfloat16())
    for n in (0, -1, 2 ** 32 + 64):  # (as a C int the last one is 64)
        with pytest.raises(ValueError):
            cache.attend(0, x, pos, n)
    with pytest.raises(ValueError):
        cache.store(0, x[:, :1].expand(2, 2 ** 32 + 1, 2, 128), x[:, :1].expand(2, 2 ** 32 + 1, 2, 128), pos)
    with pytest.raises(ValueError):
        cache.load(0, pos)
    with pytest.raises(ValueError):
        Kv8Cache(cache.k, cache.v, cache.k_scale, cache.v_scale[:, :1])


def test_graph_and_streams(torch):
    """store + attend captured once and replayed with other contents, two graphs in turn, on a side stream."""
    from work_llm_accelerator_amd.kv8 import Kv8Cache

    rng = np.random.default_rng(31)
    side = torch.cuda.Stream()
    made = []
    for seed in (1, 2):
        cache = filled(torch, 3, 40, 2, 128, seed)
        k, v, q = (torch.zeros(3, 2, h, 128, device="cuda") for h in (2, 2, 12))
        pos = ints(torch, [0, 0, 0])
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                cache.store(0, k, v, pos)
                cache.attend(0, q, pos, 2560)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            cache.store(0, k, v, pos)
            out = cache.attend(0, q, pos, 2560)
        made.append((cache, k, v, q, pos, graph, out))
    for turn in range(4):
        cache, k, v, q, pos, graph, out = made[turn % 2]
        for t in (k, v, q):
            t.copy_(torch.from_numpy(rng.standard_normal(tuple(t.shape)).astype(np.float32)))
        pos.copy_(ints(torch, [int(rng.integers(0, 2500)), -1, 2558]))
        plain = Kv8Cache(*(t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)))
        graph.replay()
        torch.cuda.synchronize()
        plain.store(0, k, v, pos)
        want = plain.attend(0, q, pos, 2560)
        assert torch.equal(out, want)
        for n in ("k", "v", "k_scale", "v_scale"):
            assert torch.equal(getattr(cache, n), getattr(plain, n))
