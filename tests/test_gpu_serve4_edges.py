"""Serving from a cache held in 4 bits at its edges."""
import math

import numpy as np
import pytest
import torch

import pagedkv
import serve4_ref as ref
from test_gpu_serve4 import HALF, PROMPT_WEIGHT, TD, Case, host, i32, prompt_case, prompt_check, typed

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# rows into the pool
# ---------------------------------------------------------------------------
def test_groups_whose_offset_rounds_above_them(gpu):
    """f16(0.3) is above 0.3: the step is negative, and codes are 0."""
    x = np.full((16, 1, 64), np.float32(0.3), np.float64)
    x[:, 0, 32:] += np.arange(32) * 1e-6
    k, x = typed(x, "f32", gpu)
    c, m, s = ref.quantize(x)
    assert np.all(m > x.max()) and np.all(s < 0) and not c.any()
    cache = pagedkv.PagedKvCache(1, 1, 16, 1, 64, pagedkv.Q4)
    slots = i32(np.arange(16), gpu)
    cache.layer(0).q4_append(k, k, slots)
    for which in (pagedkv.K, pagedkv.V):
        want = ref.chunk_bytes(which == pagedkv.K, c[:, 0], m[:, 0], s[:, 0], 16)
        assert np.array_equal(cache.read_bytes(0, which).reshape(-1), want)
    for o in cache.layer(0).q4_gather(slots):
        assert np.array_equal(host(o), np.broadcast_to(m[..., :1], o.shape))


# ---------------------------------------------------------------------------
# packed prompt attention
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dt,hd", [("f32", 64), ("f32", 128), ("f32", 256), ("f16", 64), ("f16", 128),
                                   ("bf16", 64), ("bf16", 128), ("bf16", 256)])
@pytest.mark.parametrize("others", [0, 150])
def test_prompts_see_nothing_behind_a_token(gpu, dt, hd, others):
    """Values that are not finite reach their own token and later ones only, in their own
    channels: a weight of 0 behind a token is no product.  A key's NaN reaches all of them.
    (150 more prompts: waves have units of their own.)"""
    lens = [3, 70, 33, 128, 1] + [64] * others
    q, k, v, cu, (qx, kx, vx) = prompt_case(gpu, 26, dt, 8, 2, hd, lens)
    for s, at, ch, x in [(0, 2, 0, math.nan), (1, 40, 5, math.inf), (1, 69, hd - 1, -math.inf),
                         (1, 12, 17, math.nan), (2, 32, 3, math.nan), (3, 0, 9, math.inf),
                         (3, 95, 33, math.nan), (3, 96, 33, math.inf), (4, 0, 2, math.nan)]:
        v[cu[s] + at, 1, ch] = x
        vx[cu[s] + at, 1, ch] = x
    for s, at in [(1, 50), (2, 31), (3, 100)]:
        k[cu[s] + at, 0, 1] = math.nan
        kx[cu[s] + at, 0, 1] = math.nan
    results = []
    for out_dt in {dt, "f32"}:
        out = pagedkv.prompt_attention(q, k, v, i32(cu, gpu), max_len=128, out_dtype=TD[out_dt])
        results.append((out_dt, host(out).reshape(-1, 8, hd)))
    for a, b in zip(cu[:6], cu[1:]):
        with np.errstate(invalid="ignore"):
            want, *abc = ref.attention(qx[a:b], kx[a:b], vx[a:b], b - a, hd ** -0.5)
        odd = ~np.isfinite(want)
        kv = [np.where(np.isfinite(x[a:b]), x[a:b], 0.0) for x in (kx, vx)]
        _, *abc = ref.attention(qx[a:b], *kv, b - a, hd ** -0.5)
        for out_dt, got in results:
            assert np.array_equal(got[a:b][odd], want[odd], equal_nan=True)
            tol = ref.tolerance(np.where(odd, 0.0, want), *abc, b - a, hd, PROMPT_WEIGHT[dt],
                                HALF[out_dt])
            err = np.abs(np.where(odd, 0.0, got[a:b]) - np.where(odd, 0.0, want))
            assert np.all(err <= tol), (out_dt, a, b, float((err / tol).max()))


@pytest.mark.parametrize("dt,h,kv,hd", [("bf16", 16, 8, 128), ("f16", 32, 2, 64), ("f32", 40, 2, 256),
                                        ("f32", 32, 2, 128), ("bf16", 16, 2, 256)])
def test_longer_prompts_of_waves_with_units_of_their_own(gpu, dt, h, kv, hd):
    """Hundreds of keys a unit, groups of units that a workgroup takes one after another
    because the bound is too small, and rows of no prompt that hold anything."""
    lens, lead, tail = [700, 513, 1, 330, 0, 645], 5, 9
    lens = lens + [97] * (60 if dt == "f32" else 20)
    q, k, v, cu, xs = prompt_case(gpu, 27, dt, h, kv, hd, lens, lead, tail)
    for x in (q, k, v):
        x[:lead], x[-tail:] = math.nan, math.inf
    for max_len in (700, 400):
        out = torch.full((q.shape[0], h * hd), 7.0, dtype=TD[dt], device=gpu)
        pagedkv.prompt_attention(q, k, v, i32(cu, gpu), max_len=max_len, out=out)
        prompt_check(out, cu[:9], xs, dt, hd ** -0.5)
        assert torch.all(out[:lead] == 7) and torch.all(out[-tail:] == 7)


def test_many_short_prompts_beside_a_bound_far_above_them(gpu):
    """Without max_len and with offsets on the device the bound is all rows: more
    workgroups than a launch has, of which each then takes several shares."""
    lens = [1] * 4000 + [700, 90] + [2] * 3700
    q, k, v, cu, xs = prompt_case(gpu, 28, "f16", 32, 32, 64, lens)
    out = pagedkv.prompt_attention(q, k, v, i32(cu, gpu))
    prompt_check(out, cu[3990:4020], xs, "f16", 0.125)


# ---------------------------------------------------------------------------
# attention over the pool
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_single_tokens_beside_a_long_chunk(gpu, dt):
    """The bound of a chunk is one of every sequence: what the launches are made of is
    far below sequences times it."""
    n, m = 2048, 1100
    rng = np.random.default_rng(41)
    ctx, q_lens = rng.integers(1, 20, n).tolist(), [1] * n
    ctx[100], q_lens[100] = m + 3, m
    ctx[n - 1], q_lens[n - 1] = 37, 30
    c = Case(gpu, 41, dt, 32, 8, 64, 16, ctx, q_lens)
    out = c.run()
    c.cache.check()
    some = [0, 1, 99, 101, 102, 1999, n - 2, n - 1]
    c.check(out, skip=set(range(n)) - set(some) - {100})
    # without a bound on the host
    again = c.pool.q4_attention(c.q, i32(c.tables, gpu), i32(c.ctx, gpu), cu_q_lens=i32(c.cu, gpu))
    c.cache.check()
    c.check(again, skip=set(range(n)) - set(some))


def test_bounds_may_be_far_above_the_rows(gpu):
    c = Case(gpu, 42, "bf16", 8, 2, 64, 16, [40, 5], [30, 1])
    for most in (31, 1 << 20, 1 << 30):
        c.check(c.run(max_q_len=most))
    c.check(c.run(max_q_len=1 << 30, max_context_len=1 << 20))


@pytest.mark.parametrize("kind", [0, 1])
def test_scratch_of_chunks_is_small(gpu, kind):
    """A call's scratch holds partial results of single tokens' and short contexts' parts,
    not of every row of long chunks."""
    cache = pagedkv.PagedKvCache(1, 1, 16, 8, 128, pagedkv.Q4)
    size = pagedkv.lib().pkv_q4_workspace_bytes
    if kind == 0:  # 12 chunks, 1200 rows: one row of a sequence may have parts, 8 of them (96
        # workgroups without, 768 wanted)
        assert size(cache.handle, 12, 1200, 600, 8200, 64) <= 12 * 64 * 8 * 130 * 4
    else:  # 255 single tokens and 8192 rows: two rows of a sequence, 32 parts
        assert size(cache.handle, 256, 8447, 8192, 131072, 32) <= 256 * 2 * 32 * 32 * 130 * 4


@pytest.mark.parametrize("h,kv,hd", [(8, 2, 128), (4, 2, 64), (4, 4, 256)])
def test_f32_chunks_over_long_contexts(gpu, h, kv, hd):
    """Chunks of f32 queries that fill the GPU go through all keys in one part, past the
    4096 whose block ids a wave has at once."""
    c = Case(gpu, 44, "f32", h, kv, hd, 16, [9003] + [40] * 30, [40] * 31)
    out = c.run(max_q_len=800)
    c.cache.check()
    c.check(out, skip=range(2, 31))


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("h,kv,hd", [(32, 8, 64), (32, 8, 128), (16, 8, 256)])
def test_queries_with_far_out_channels(gpu, dt, h, kv, hd):
    """One channel of each group 64 times the others.  Scores have a deviation of some 2.5,
    so scale q is at most 2.5 / sqrt(groups) there.  Products with codes are kept to 2^-17 of
    the largest of eight: the seven beside that channel are off by 2^-17 sqrt(7 / 12) of it at
    random, times a step of the keys, 0.3, and 2.5 over all groups: 2^-17.8 in a score.
    Values' sums of 2000 keys, of which some four matter, lose 2^-20: 2^-17 in norm."""
    c = Case(gpu, h + hd, dt, h, kv, hd, 16, [2000], [1], scale=2.5 / 64 / math.sqrt(hd // 32))
    k, v = c.rng.normal(size=(2, c.cache.num_blocks * 16, kv, hd))
    k, kx = typed(k.astype(np.float32), dt, gpu)
    v, vx = typed(v.astype(np.float32), dt, gpu)
    c.pool.q4_append(k, v, torch.arange(len(k), dtype=torch.int32, device=gpu))
    c.take(kx, vx)
    q = c.rng.normal(size=(1, h, hd))
    q[..., ::32] *= 64.0
    c.q, c.qx = typed(q, dt, gpu)
    want = ref.attention(c.qx, *c.rows(0)[0], 1, c.scale, *c.rows(0)[1])[0]
    got = host(c.run(out_dtype=torch.float32)).reshape(want.shape)
    off = np.linalg.norm(got - want) / np.linalg.norm(want)
    assert off <= 2.0 ** -17, math.log2(off)


@pytest.mark.parametrize("dt,h,kv,hd", [("bf16", 8, 2, 128), ("f16", 7, 1, 64), ("f32", 8, 2, 64)])
def test_more_parts_than_lanes(gpu, dt, h, kv, hd):
    """A sequence in 66 parts and more: the join goes through them 64 at a time."""
    c = Case(gpu, 43, dt, h, kv, hd, 16, [20001, 17000, 5])
    c.check(c.run())
    c.check(c.run(max_context_len=1 << 20))


# ---------------------------------------------------------------------------
# streams
# ---------------------------------------------------------------------------
def test_another_stream_changes_no_refusal(gpu):
    side = torch.cuda.Stream()
    x = torch.zeros((2, 100), device=gpu)
    toks, cu, cpu = i32([1, 2], gpu), i32([0, 1, 2], gpu), torch.tensor([0, 1, 2], dtype=torch.int32)
    rows = torch.zeros((4, 2, 64), device=gpu, dtype=torch.float16)
    pool = pagedkv.PagedKvCache(1, 2, 16, 2, 64, pagedkv.Q4).layer(0)
    for s in (None, side):
        for bad in (cpu, [0, 1, 2]):
            with pytest.raises(ValueError, match="cu_tokens must be a tensor on"):
                pagedkv.adjust_logits(x, tokens=toks, cu_tokens=bad, stream=s)
        with pytest.raises(ValueError, match="out must be"):
            pagedkv.adjust_logits(x, out=x.cpu(), stream=s)
        with pytest.raises(ValueError, match="k must be a tensor on"):
            pagedkv.prompt_attention(rows, rows.cpu(), rows, [0, 4], stream=s)
        with pytest.raises(ValueError, match="out must be"):
            pagedkv.prompt_attention(rows, rows, rows, [0, 4], out=torch.zeros((4, 128)), stream=s)
        with pytest.raises(ValueError, match="v must be a tensor on"):
            pool.q4_append(rows, rows.cpu(), [0, 1, 2, 3], stream=s)
    got = pagedkv.adjust_logits(x, tokens=toks, cu_tokens=cu, stream=side)
    side.synchronize()
    assert not got.any()
