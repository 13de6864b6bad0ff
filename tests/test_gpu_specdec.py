"""Speculative decoding over long contexts on the GPU: step tables, key
bounds, the choice of blocks, attention over them and draft verification,
each against its plain 64-bit implementation (specdec_ref), then together."""
import numpy as np
import pytest
import torch

import pagedkv
import specdec_ref as ref
from pagedkv import workload as wl

pytestmark = pytest.mark.gpu

TD = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODE = {"f32": wl.F32, "f16": wl.F16, "bf16": wl.BF16}


def i32(x, gpu):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=gpu)


def host(t):
    return t.cpu().numpy().astype(np.int64)


def rounded(x, dt):
    """float64 values of x rounded to the type."""
    return torch.tensor(x).to(TD[dt]).double().numpy()


def to_pool(dt, k, v, bs):
    """A one-layer pool holding k, v of (num_blocks, bs, kv, hd)."""
    nb, _, kv, hd = k.shape
    cache = pagedkv.PagedKvCache(1, nb, bs, kv, hd, TD[dt])
    pool = cache.layer(0)
    slots = torch.arange(nb * bs, dtype=torch.int32, device=cache.device)
    kk, vv = (torch.tensor(x).to(TD[dt]).to(cache.device).reshape(nb * bs, kv, hd) for x in (k, v))
    pool.append(kk, vv, slots)
    torch.cuda.synchronize()
    return cache, pool


def place(rng, ctx, bs, spare=3, width=None):
    """Block tables of disjoint random blocks; (tables, blocks of the pool)."""
    need = [-(-int(c) // bs) for c in ctx]
    nb = sum(need) + spare
    perm = rng.permutation(nb)
    tables = np.zeros((len(ctx), max(max(need), width or 1)), np.int64)
    at = 0
    for i, n in enumerate(need):
        tables[i, :n] = perm[at:at + n]
        at += n
    return tables, nb, perm[at:]


# ---------------------------------------------------------------------------
# step tables
# ---------------------------------------------------------------------------
def step_case(seed, n, bs, width, hi, new_hi, extra=2):
    rng = np.random.default_rng(seed)
    seq = rng.integers(0, hi + 1, n)
    new = rng.integers(0, new_hi + 1, n)
    have = np.minimum(-(-seq // bs) + rng.integers(0, 3, n), width)
    total = np.maximum(have, -(-(seq + new) // bs))
    nb = int(total.sum()) + extra + 7
    perm = rng.permutation(nb)
    tables = rng.integers(0, nb, (n, width))
    at = 0
    for i in range(n):
        tables[i, :have[i]] = perm[at:at + have[i]]
        at += have[i]
    return seq, new, tables, have, perm[at:], nb


def run_step(gpu, seq, new, tables, have, free, count, bs, nb, tokens, **kw):
    r = pagedkv.step_tables(i32(seq, gpu), i32(new, gpu), i32(tables, gpu), i32(have, gpu),
                            i32(free, gpu), i32([count], gpu), bs, nb, tokens, **kw)
    torch.cuda.synchronize()
    return r


def same_step(r, want):
    for name, w in want.items():
        assert np.array_equal(host(getattr(r, name)), w), name


@pytest.mark.parametrize("n,bs,width,hi,new_hi,pad", [
    (1, 16, 1, 0, 1, 0), (1, 16, 64, 900, 40, 3), (7, 16, 64, 900, 5, 3), (64, 1, 50, 40, 9, 0),
    (300, 16, 33, 400, 60, 11), (5, 256, 9, 1900, 300, 1), (3, 32, 2000, 60000, 3000, 100),
    (1100, 8, 7, 40, 16, 5), (17, 16, 20, 250, 0, 4), (2, 64, 70, 4000, 400, 0)])
def test_step_tables(gpu, n, bs, width, hi, new_hi, pad):
    a = step_case(n * 7 + bs, n, bs, width, min(hi, width * bs - new_hi), new_hi)
    seq, new, tables, have, free, nb = a
    tokens = int(new.sum()) + pad
    want = ref.step_tables(seq, new, tables, have, free, len(free), bs, nb, tokens)
    assert want["status"][0] == 0
    same_step(run_step(gpu, *a[:5], len(free), bs, nb, tokens), want)
    # a free list that is longer than its count
    used = len(free) - 2
    want = ref.step_tables(seq, new, tables, have, free, used, bs, nb, tokens)
    same_step(run_step(gpu, *a[:5], used, bs, nb, tokens), want)


@pytest.mark.parametrize("what", ["short", "negative", "narrow", "tokens", "count", "have", "negnew"])
def test_step_tables_that_cannot_be_built_change_nothing(gpu, what):
    seq, new, tables, have, free, nb = step_case(11, 9, 16, 12, 100, 20)
    new[2] = 25
    have[2] = -(-seq[2] // 16)
    count, tokens = len(free), int(new.sum()) + 2
    if what == "short":
        count = 1
    elif what == "negative":
        seq[4] = -3
    elif what == "narrow":
        new[8] = 16 * 12 + 1 - seq[8]
    elif what == "tokens":
        tokens = int(new.sum()) - 1
    elif what == "count":
        count = len(free) + 1
    elif what == "have":
        have[3] = 13
    else:
        new[0] = -1
    want = ref.step_tables(seq, new, tables, have, free, count, 16, nb, tokens)
    assert want["status"][0] == (-1 if what != "short" else want["status"][0]) != 0
    same_step(run_step(gpu, seq, new, tables, have, free, count, 16, nb, tokens), want)


def test_step_tables_bad_ids_and_empty_step(gpu):
    seq, new, tables, have, free, nb = step_case(12, 4, 16, 12, 100, 20)
    new[:] = 18
    free[-1], tables[1, 0] = nb + 5, -1
    seq[1], have[1] = 0, 1
    tokens = 80
    want = ref.step_tables(seq, new, tables, have, free, len(free), 16, nb, tokens)
    assert (want["slot_mapping"] == 2 ** 31 - 1).any()
    same_step(run_step(gpu, seq, new, tables, have, free, len(free), 16, nb, tokens), want)
    z = np.zeros(0, np.int64)
    r = run_step(gpu, z, z, np.zeros((0, 3), np.int64), z, free, 3, 16, nb, 5)
    assert host(r.cu_q_lens).tolist() == [0] and host(r.status).tolist() == [0]
    assert host(r.free_count).tolist() == [3] and (host(r.slot_mapping) == -1).all()


def test_step_tables_in_place_on_the_table_array(gpu):
    seq, new, tables, have, free, nb = step_case(13, 40, 16, 30, 400, 40)
    tokens = int(new.sum())
    want = ref.step_tables(seq, new, tables, have, free, len(free), 16, nb, tokens)
    d = [i32(x, gpu) for x in (seq, new, tables, have, free, [len(free)])]
    o = [torch.empty(k, dtype=torch.int32, device=gpu) for k in (40, 1, 40, 41, tokens, tokens, 1)]
    p = [t.data_ptr() for t in d]
    rc = pagedkv.lib().pkv_step_tables(16, nb, p[0], p[1], 40, p[2], p[3], 30, p[4], len(free), p[5],
                                       tokens, p[2], *[t.data_ptr() for t in o], None)
    assert rc == 0
    torch.cuda.synchronize()
    got = pagedkv.StepTables(d[2], o[0], o[1], o[2], o[3], o[4], o[5], o[6])
    same_step(got, want)


# ---------------------------------------------------------------------------
# key bounds
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dt,kv,hd,bs", [("bf16", 8, 128, 16), ("f16", 2, 64, 16), ("f32", 2, 64, 4),
                                         ("f32", 1, 256, 32), ("bf16", 3, 256, 1),
                                         ("f16", 1, 128, 256), ("bf16", 5, 64, 64)])
def test_key_bounds(gpu, dt, kv, hd, bs):
    rng = np.random.default_rng(kv * hd + bs)
    ctx = np.array([1, bs, bs + 1, 5 * bs - 1, 7 * bs, 3, 0, 2 * bs + bs // 2 + 1])
    first = np.array([0, 0, 0, 2 * bs, 7 * bs - 1, 3, 0, bs])
    tables, nb, rest = place(rng, ctx, bs)
    k = rounded(rng.normal(size=(nb, bs, kv, hd)), dt)
    for s, c in enumerate(ctx):  # keys past a context may be anything
        if c % bs:
            k[tables[s, c // bs], c % bs:] = np.nan
    cache, pool = to_pool(dt, k, k, bs)
    bounds = pool.new_key_bounds()
    bounds += 7.0
    got = pool.update_key_bounds(bounds, tables, ctx, first, 5 * bs)
    want = ref.key_bounds(np.full((nb, kv, 2, hd), 7.0), k, tables, first, ctx, bs)
    torch.cuda.synchronize()
    cache.check()
    assert got is bounds and np.array_equal(bounds.double().cpu().numpy(), want)  # exact
    # all blocks, from lengths alone
    pool.update_key_bounds(bounds, tables, ctx)
    want = ref.key_bounds(want, k, tables, np.zeros_like(first), ctx, bs)
    torch.cuda.synchronize()
    cache.check()
    assert np.array_equal(bounds.double().cpu().numpy(), want)
    cache.close()


@pytest.mark.parametrize("what", ["block", "length", "long", "first"])
def test_key_bounds_reports_bad_data(gpu, what):
    rng = np.random.default_rng(2)
    ctx, first, bs = np.array([40, 50, 33]), np.array([30, 49, 0]), 16
    tables, nb, _ = place(rng, ctx, bs)
    k = rounded(rng.normal(size=(nb, bs, 2, 64)), "bf16")
    cache, pool = to_pool("bf16", k, k, bs)
    want = ref.key_bounds(np.zeros((nb, 2, 2, 64)), k, tables[[0, 2]], first[[0, 2]], ctx[[0, 2]], bs)
    if what == "block":
        tables[1, 3] = nb
    elif what == "length":
        ctx[1] = 16 * tables.shape[1] + 1
    elif what == "long":
        first[1] = 10
    else:
        first[1] = -1
    bounds = pool.update_key_bounds(pool.new_key_bounds(), tables, ctx, first, 34)
    with pytest.raises(pagedkv.PagedKvError):
        cache.check()
    assert np.array_equal(bounds.double().cpu().numpy(), want)
    cache.close()


# ---------------------------------------------------------------------------
# choice of blocks
# ---------------------------------------------------------------------------
def make_bounds(rng, nb, kv, hd, dt, near=False):
    """Bounds of blocks around centres; near: of almost equal scores."""
    mid = rng.normal(size=(nb, kv, hd)) * 0.7
    half = np.abs(rng.normal(size=(nb, kv, hd))) * 0.4 + 1.0
    if near:
        mid = np.repeat(mid[:1], nb, 0)
        half = np.repeat(half[:1], nb, 0)
        mid[:, :, 0] *= 1 + rng.integers(0, 9, (nb, kv)) * 2.0 ** -8
    return rounded(np.stack((mid - half, mid + half), 2), dt)


def run_select(gpu, dt, q, bounds, tables, cu, ctx, bs, top, first, last, check=True, **kw):
    nb, kv, _, hd = bounds.shape
    cache = pagedkv.PagedKvCache(1, nb, bs, kv, hd, TD[dt])
    out = cache.layer(0).select_blocks(
        torch.tensor(q).to(TD[dt]).to(gpu), torch.tensor(bounds).to(TD[dt]).to(gpu), tables, ctx,
        top, first, last, cu_q_lens=None if cu is None else i32(cu, gpu), **kw)
    torch.cuda.synchronize()
    if check:
        cache.check()
    cache.close()
    return host(out)


@pytest.mark.parametrize("dt,H,kv,hd,bs,top,first,last,near", [
    ("bf16", 32, 8, 128, 16, 20, 1, 2, False), ("f16", 8, 8, 64, 16, 11, 0, 1, False),
    ("f32", 14, 2, 64, 16, 30, 2, 3, False), ("bf16", 16, 8, 128, 16, 7, 1, 1, True),
    ("f16", 12, 4, 256, 4, 25, 1, 4, True), ("f32", 4, 1, 128, 1, 50, 3, 1, True),
    ("bf16", 20, 1, 64, 32, 9, 0, 2, False), ("f16", 16, 1, 128, 8, 33, 1, 1, True),
    ("f32", 40, 2, 256, 16, 12, 1, 2, True), ("bf16", 6, 2, 64, 256, 3, 1, 2, False)])
def test_select(gpu, dt, H, kv, hd, bs, top, first, last, near):
    rng = np.random.default_rng(H * hd + bs)
    ctx = np.array([1, top * bs, top * bs + 1, 37 * bs + 1, 111 * bs, 0, (top + 1) * bs, 150 * bs - 1])
    tables, nb, _ = place(rng, ctx, bs)
    bounds = make_bounds(rng, nb, kv, hd, dt, near)
    q = rounded(rng.normal(size=(len(ctx), H, hd)), dt)
    want = ref.select(q, bounds, tables, None, ctx, bs, top, first, last)
    assert np.array_equal(run_select(gpu, dt, q, bounds, tables, None, ctx, bs, top, first, last), want)


@pytest.mark.parametrize("dt,H,kv,hd,near", [("bf16", 32, 8, 128, False), ("f16", 8, 4, 64, True),
                                             ("f32", 14, 2, 64, False), ("bf16", 3, 3, 64, False),
                                             ("bf16", 48, 2, 64, True)])
def test_select_for_chunks(gpu, dt, H, kv, hd, near):
    rng = np.random.default_rng(H + hd)
    bs, top = 16, 14
    m = np.array([1, 5, 0, 3, 17, 2])
    ctx = np.array([900, 16 * 14 + 3, 50, 2, 1500, 16 * 15])  # (rows of no key in the fourth)
    cu = np.concatenate(([0], np.cumsum(m)))
    tables, nb, _ = place(rng, ctx, bs)
    bounds = make_bounds(rng, nb, kv, hd, dt, near)
    q = rounded(rng.normal(size=(cu[-1], H, hd)), dt)
    want = ref.select(q, bounds, tables, cu, ctx, bs, top, 1, 2)
    assert np.array_equal(run_select(gpu, dt, q, bounds, tables, cu, ctx, bs, top, 1, 2), want)
    assert np.array_equal(run_select(gpu, dt, q, bounds, tables, cu, ctx, bs, top, 1, 2,
                                     max_q_len=17, max_context_len=1500), want)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_key_bounds_pass_over_nan(gpu, dt):
    # an element that is NaN in some keys of a block, in all of them, and infinite ones
    rng = np.random.default_rng(5)
    bs, kv, hd = 16, 2, 64
    k = rounded(rng.normal(size=(3, bs, kv, hd)), dt)
    k[0, 3:9, 1, 7] = np.nan
    k[1, :, 0, 5] = np.nan
    k[2, 4, 1, 2], k[2, 5, 1, 2] = np.inf, -np.inf
    cache, pool = to_pool(dt, k, k, bs)
    bounds = pool.update_key_bounds(pool.new_key_bounds(), i32([[0, 1, 2]], gpu), i32([48], gpu))
    cache.check()
    want = np.stack([np.fmin.reduce(k, axis=1), np.fmax.reduce(k, axis=1)], axis=2)
    want[1, 0, 0, 5], want[1, 0, 1, 5] = np.inf, -np.inf
    assert np.array_equal(bounds.double().cpu().numpy(), want)
    cache.close()


@pytest.mark.parametrize("what", ["zero", "equal", "inf", "nan", "query", "huge", "negative"])
def test_select_ties_and_values_that_are_not_finite(gpu, what):
    rng = np.random.default_rng(4)
    dt, H, kv, hd, bs, top = "f32" if what == "huge" else "bf16", 8, 2, 64, 16, 12
    ctx = np.array([100 * bs - 3, 60 * bs, 30 * bs + 1])
    tables, nb, _ = place(rng, ctx, bs)
    bounds = make_bounds(rng, nb, kv, hd, dt)
    q = rounded(rng.normal(size=(3, H, hd)), dt)
    if what == "zero":
        q[1] = 0.0
    elif what == "equal":
        bounds[:] = bounds[:1]
    elif what == "inf":
        bounds[tables[0, 70], 1, 1, 3] = np.inf
        bounds[tables[0, 20], 0, 0, 5] = -np.inf
    elif what == "nan":
        bounds[tables[1, 33:50], 1, :, 3] = np.nan
    elif what == "query":
        q[2, 5, 7] = np.inf
    elif what == "huge":
        bounds[tables[0, 10:40]] *= 1e37
        q[0] *= 10.0
    else:  # every score far below zero: a zero-filled tile must not win
        bounds = rounded(-np.abs(bounds) * np.sign(q[0].reshape(2, 4, 64)[:, :1, None])[:, 0], dt)
        bounds = np.stack((bounds.min(2), bounds.max(2)), 2)
    if what == "huge":  # past the f32 range: +inf
        b, x = bounds.astype(np.float32), q.astype(np.float32)
        want = []
        for s, n in enumerate((100, 60, 31)):
            sc = ref.block_scores(q[s], bounds, tables[s], n)
            sc = np.where(np.abs(sc) > np.finfo(np.float32).max, np.inf, sc)
            rows = []
            for g in range(kv):
                mid = np.arange(1, n - 2)
                best = mid[np.argsort(-sc[g, mid], kind="stable")[:9]]
                rows.append(np.sort(np.concatenate(([0], best, [n - 2, n - 1]))))
            want.append(rows)
        want = np.array(want)
    else:
        want = ref.select(q, bounds, tables, None, ctx, bs, top, 1, 2)
    assert np.array_equal(run_select(gpu, dt, q, bounds, tables, None, ctx, bs, top, 1, 2), want)


def test_select_scores_at_the_end_of_the_f32_range(gpu):
    # blocks that are not finite rank first also where the border between taken
    # and left blocks plus its error bound is past the largest float
    kv, hd, bs, top, n = 2, 64, 16, 12, 100
    rng = np.random.default_rng(12)
    ctx = np.array([n * bs, n * bs])
    tables, nb, _ = place(rng, ctx, bs)
    bounds = np.zeros((nb, kv, 2, hd))
    big = float(np.float32(3.4028e38))
    bounds[:, :, 1, 0] = 1e38
    # want is 9: six blocks at the range's end and five that are not finite
    bounds[tables[:, 20:32:2], :, 1, 0] = big
    bounds[tables[:, [50, 60, 70]], :, 0, 5] = np.nan
    bounds[tables[:, [80, 90]], :, 1, 9] = np.inf
    q = np.zeros((2, 4, hd))
    q[:, :, 0] = 1.0
    want = ref.select(q, bounds, tables, None, ctx, bs, top, 1, 2)
    assert set([50, 60, 70, 80, 90]) < set(want[0, 0])
    assert np.array_equal(run_select(gpu, "f32", q, bounds, tables, None, ctx, bs, top, 1, 2), want)


def test_select_more_blocks_than_fit_in_lds(gpu):
    rng = np.random.default_rng(6)
    ctx = np.array([20000, 9000])
    tables, nb, _ = place(rng, ctx, 1)
    bounds = make_bounds(rng, nb, 1, 64, "bf16")
    q = rounded(rng.normal(size=(2, 2, 64)), "bf16")
    want = ref.select(q, bounds, tables, None, ctx, 1, 700, 5, 30)
    assert np.array_equal(run_select(gpu, "bf16", q, bounds, tables, None, ctx, 1, 700, 5, 30), want)


def test_select_reports_bad_data_and_leaves_other_rows(gpu):
    rng = np.random.default_rng(8)
    bs, top, ctx = 16, 6, np.array([400, 500])
    tables, nb, _ = place(rng, ctx, bs)
    bounds = make_bounds(rng, nb, 2, 64, "f16")
    q = rounded(rng.normal(size=(5, 4, 64)), "f16")
    cu = np.array([0, 1, 3])  # rows 3 and 4 belong to no sequence
    cache = pagedkv.PagedKvCache(1, nb, bs, 2, 64, torch.float16)
    out = torch.full((5, 2, top), -7, dtype=torch.int32, device=gpu)
    args = [torch.tensor(x).half().to(gpu) for x in (q, bounds)]
    pool = cache.layer(0)
    pool.select_blocks(*args, tables, ctx, top, 1, 1, cu_q_lens=cu, max_q_len=2, out=out)
    cache.check()
    assert np.array_equal(host(out)[:3], ref.select(q, bounds, tables, cu, ctx, bs, top, 1, 1))
    assert (host(out)[3:] == -7).all()
    # a chunk beyond max_q_len, a context beyond max_context_len, a bad block
    pool.select_blocks(*args, tables, ctx, top, 1, 1, cu_q_lens=cu, max_q_len=1)
    with pytest.raises(pagedkv.PagedKvError):
        cache.check()
    pool.select_blocks(*args, tables, ctx, top, 1, 1, cu_q_lens=cu, max_q_len=2, max_context_len=450)
    with pytest.raises(pagedkv.PagedKvError):
        cache.check()
    tables[1, 4] = nb + 3
    pool.select_blocks(*args, tables, ctx, top, 1, 1, cu_q_lens=cu, max_q_len=2)
    with pytest.raises(pagedkv.PagedKvError):
        cache.check()
    cache.close()


# ---------------------------------------------------------------------------
# attention over chosen blocks
# ---------------------------------------------------------------------------
def choose(rng, rows, kv, top, bs, how):
    """Lists for rows of (sequence, keys): distinct blocks of the context."""
    out = np.full((len(rows), kv, top), -1, np.int64)
    for r, (_, keys) in enumerate(rows):
        nb = -(-keys // bs)
        for g in range(kv):
            pick = rng.permutation(nb)[:rng.integers(0, top + 1) if how == "holes" else top]
            if nb and how == "select" and nb - 1 not in pick:
                pick[0] = nb - 1
            if how == "select":
                out[r, g, :len(pick)] = np.sort(pick)
            else:  # any order, entries anywhere
                out[r, g, rng.permutation(top)[:len(pick)]] = pick
    return out


def run_sparse(gpu, dt, cache, pool, q, blocks, tables, cu, ctx, **kw):
    out = pool.sparse_attention(torch.tensor(q).to(TD[dt]).to(gpu), i32(blocks, gpu), tables, ctx,
                                cu_q_lens=None if cu is None else i32(cu, gpu), **kw)
    torch.cuda.synchronize()
    cache.check()
    return out.double().cpu().numpy().reshape(q.shape)


def within(got, want, bound, out_dt):
    half = 0.0 if out_dt == "f32" else torch.finfo(TD[out_dt]).eps / 2
    err = np.abs(got - want)
    tol = bound + (half + 2.0 ** -24) * (np.abs(want) + bound)
    if out_dt == "f16":
        tol = tol + 2.0 ** -25  # half a step of its smallest values
    assert np.isfinite(got).all() and (err <= tol).all(), (err - tol).max()


@pytest.mark.parametrize("how", ["select", "holes"])
@pytest.mark.parametrize("dt,H,kv,hd,bs,top,out_dt", [
    ("bf16", 32, 8, 128, 16, 20, "bf16"), ("bf16", 8, 1, 128, 16, 70, "f32"),
    ("f16", 8, 8, 64, 16, 5, "f32"), ("f32", 14, 2, 64, 16, 9, "f32"),
    ("f16", 32, 2, 128, 32, 40, "f16"), ("bf16", 2, 2, 256, 4, 33, "f32"),
    ("f32", 6, 3, 128, 1, 100, "f32"), ("bf16", 20, 1, 64, 8, 12, "bf16"),
    ("f16", 10, 2, 256, 256, 3, "f32"), ("f32", 16, 1, 256, 64, 4, "f32"),
    ("bf16", 4, 2, 64, 2, 1, "f32"), ("f16", 4, 1, 64, 128, 20, "f32")])
def test_sparse_attention(gpu, dt, H, kv, hd, bs, top, out_dt, how):
    rng = np.random.default_rng(H * hd + bs + len(how))
    ctx = np.array([1, bs, 3 * bs - 1, 90 * bs + 1, 0, top * bs, 2, 41 * bs])
    tables, nb, rest = place(rng, ctx, bs)
    k, v = (rounded(rng.normal(size=(nb, bs, kv, hd)), dt) for _ in range(2))
    for s, c in enumerate(ctx):  # what lies behind a context must not matter
        if c % bs:
            k[tables[s, c // bs], c % bs:] = np.nan
            v[tables[s, c // bs], c % bs:] = np.nan
    k[rest], v[rest] = np.nan, np.inf
    cache, pool = to_pool(dt, k, v, bs)
    q = rounded(rng.normal(size=(len(ctx), H, hd)) * 1.5, dt)
    blocks = choose(rng, ref.rows_of(None, ctx), kv, top, bs, how)
    want, bound = ref.sparse_attention(q, k, v, blocks, tables, None, ctx, bs, hd ** -0.5)
    got = run_sparse(gpu, dt, cache, pool, q, blocks, tables, None, ctx, out_dtype=TD[out_dt])
    within(got, want, bound, out_dt)
    assert (got[4] == 0).all()
    cache.close()


@pytest.mark.parametrize("dt,H,kv,hd,bs", [("bf16", 64, 8, 128, 16), ("f32", 14, 2, 64, 16),
                                           ("f16", 4, 4, 64, 4)])
def test_sparse_attention_of_chunks(gpu, dt, H, kv, hd, bs):
    rng = np.random.default_rng(H + hd)
    m, ctx = np.array([1, 6, 0, 4, 5]), np.array([700, 45, 9, 2, 300])
    cu = np.concatenate(([0], np.cumsum(m)))
    tables, nb, _ = place(rng, ctx, bs)
    k, v = (rounded(rng.normal(size=(nb, bs, kv, hd)), dt) for _ in range(2))
    cache, pool = to_pool(dt, k, v, bs)
    q = rounded(rng.normal(size=(cu[-1] + 2, H, hd)), dt)  # two rows of no sequence
    blocks = choose(rng, ref.rows_of(cu, ctx), kv, 11, bs, "select")
    blocks = np.concatenate((blocks, np.full((2, kv, 11), -1)))
    want, bound = ref.sparse_attention(q[:-2], k, v, blocks, tables, cu, ctx, bs, 0.2)
    for kw in ({}, {"max_q_len": 6}):
        out = torch.full((len(q), H * hd), 5.0, dtype=torch.float32, device=gpu)
        got = run_sparse(gpu, dt, cache, pool, q, blocks, tables, cu, ctx, scale=0.2, out=out, **kw)
        within(got[:-2], want, bound, "f32")
        assert (got[-2:] == 5.0).all()
    cache.close()


@pytest.mark.parametrize("chunks", [False, True])
@pytest.mark.parametrize("dt,H,kv,hd,bs,top,out_dt", [
    ("bf16", 8, 8, 128, 16, 30, "f32"), ("f16", 16, 8, 64, 16, 61, "f16"),
    ("bf16", 24, 8, 256, 16, 17, "bf16"), ("f16", 8, 8, 128, 8, 45, "f32"),
    ("bf16", 160, 8, 64, 32, 20, "f32"), ("f32", 8, 8, 64, 16, 30, "f32"),
    ("bf16", 24, 8, 256, 16, 16, "bf16")])
def test_sparse_attention_of_many_rows(gpu, dt, H, kv, hd, bs, top, out_dt, chunks):
    # enough (row, kv head) pairs for a workgroup each; some have few blocks or none
    rng = np.random.default_rng(hd + top)
    ctx = rng.integers(1, 2 * top * bs, 24)
    ctx[::6] = rng.integers(0, 2 * bs, 4)
    m = rng.integers(0, 4, 24) if chunks else None
    cu = np.concatenate(([0], np.cumsum(m))) if chunks else None
    tables, nb, _ = place(rng, ctx, bs)
    k, v = (rounded(rng.normal(size=(nb, bs, kv, hd)), dt) for _ in range(2))
    cache, pool = to_pool(dt, k, v, bs)
    q = rounded(rng.normal(size=(cu[-1] if chunks else 24, H, hd)), dt)
    blocks = choose(rng, ref.rows_of(cu, ctx), kv, top, bs, "holes")
    blocks[::2] = choose(rng, ref.rows_of(cu, ctx), kv, top, bs, "select")[::2]
    want, bound = ref.sparse_attention(q, k, v, blocks, tables, cu, ctx, bs, hd ** -0.5)
    got = run_sparse(gpu, dt, cache, pool, q, blocks, tables, cu, ctx, out_dtype=TD[out_dt])
    within(got, want, bound, out_dt)
    cache.close()


def test_sparse_attention_of_rows_in_sixteen_parts(gpu):
    # 21 chunk rows, 8 kv heads, 1024 tokens listed: parts of 64 in one workgroup
    rng = np.random.default_rng(77)
    bs, kv, hd, top, m = 16, 8, 64, 64, np.full(7, 3)
    ctx = rng.integers(1100, 3000, 7)
    cu = np.concatenate(([0], np.cumsum(m)))
    tables, nb, _ = place(rng, ctx, bs)
    k, v = (rounded(rng.normal(size=(nb, bs, kv, hd)), "f16") for _ in range(2))
    cache, pool = to_pool("f16", k, v, bs)
    q = rounded(rng.normal(size=(21, 16, hd)) * 2, "f16")
    blocks = choose(rng, ref.rows_of(cu, ctx), kv, top, bs, "select")
    want, bound = ref.sparse_attention(q, k, v, blocks, tables, cu, ctx, bs, hd ** -0.5)
    got = run_sparse(gpu, "f16", cache, pool, q, blocks, tables, cu, ctx, out_dtype=torch.float32,
                     max_q_len=3)
    within(got, want, bound, "f32")
    cache.close()


@pytest.mark.parametrize("dt,H,kv,hd", [("bf16", 32, 8, 128), ("f16", 7, 1, 64)])
def test_all_blocks_is_decode_and_prefill_attention(gpu, dt, H, kv, hd):
    rng = np.random.default_rng(hd)
    bs, m, ctx = 16, np.array([3, 1, 4]), np.array([200, 17, 333])
    cu = np.concatenate(([0], np.cumsum(m)))
    tables, nb, _ = place(rng, ctx, bs)
    k, v = (rounded(rng.normal(size=(nb, bs, kv, hd)), dt) for _ in range(2))
    cache, pool = to_pool(dt, k, v, bs)
    q = rounded(rng.normal(size=(cu[-1], H, hd)), dt)
    width = tables.shape[1]
    blocks = np.tile(np.arange(width), (len(q), kv, 1))
    for r, (_, keys) in enumerate(ref.rows_of(cu, ctx)):
        blocks[r, :, -(-keys // bs):] = -1
    got = run_sparse(gpu, dt, cache, pool, q, blocks, tables, cu, ctx, out_dtype=torch.float32)
    qd = torch.tensor(q).to(TD[dt]).to(gpu)
    dense = pool.prefill_attention(qd, cu, ctx, tables, 4, 333, out_dtype=torch.float32)
    _, bound = ref.sparse_attention(q, k, v, blocks, tables, cu, ctx, bs, hd ** -0.5)
    # the 16-bit prefill rounds its weights to 16 bits: one more half step of them
    half = torch.finfo(TD[dt]).eps / 2
    tol = 2 * bound + 2 * half * np.abs(v).max()
    assert (np.abs(got - dense.double().cpu().numpy().reshape(got.shape)) <= tol).all()
    lastrow = cu[1:] - 1
    one = run_sparse(gpu, dt, cache, pool, q[lastrow], blocks[lastrow], tables, None, ctx,
                     out_dtype=torch.float32)
    dec = pool.decode_attention(qd[torch.tensor(lastrow)], tables, ctx, out_dtype=torch.float32)
    assert (np.abs(one - dec.double().cpu().numpy().reshape(one.shape)) <= 2 * bound[lastrow]).all()
    cache.close()


@pytest.mark.parametrize("what", ["index", "block", "long"])
def test_sparse_attention_skips_and_reports_bad_entries(gpu, what):
    rng = np.random.default_rng(9)
    bs, ctx, H, kv, hd = 16, np.array([100, 300]), 8, 2, 64
    tables, nb, _ = place(rng, ctx, bs)
    k, v = (rounded(rng.normal(size=(nb, bs, kv, hd)), "bf16") for _ in range(2))
    cache, pool = to_pool("bf16", k, v, bs)
    q = rounded(rng.normal(size=(2, H, hd)), "bf16")
    blocks = choose(rng, ref.rows_of(None, ctx), kv, 5, bs, "select")
    good = blocks.copy()
    call_ctx, call_tables = ctx.copy(), tables.copy()
    if what == "index":
        blocks[0, 1, 2], good[0, 1, 2] = 7, -1  # one past the context's last block
    elif what == "block":
        call_tables[1, blocks[1, 0, 1]] = nb
        good[1][good[1] == blocks[1, 0, 1]] = -1
    else:
        call_ctx[1] = 16 * tables.shape[1] + 9
        ctx[1] = 16 * tables.shape[1]
    want, bound = ref.sparse_attention(q, k, v, good, tables, None, ctx, bs, hd ** -0.5)
    out = pool.sparse_attention(torch.tensor(q).bfloat16().to(gpu), i32(blocks, gpu), call_tables,
                                call_ctx, out_dtype=torch.float32)
    with pytest.raises(pagedkv.PagedKvError):
        cache.check()
    within(out.double().cpu().numpy().reshape(q.shape), want, bound, "f32")
    cache.close()


@pytest.mark.parametrize("dt,H,kv,rows", [("bf16", 4, 2, 5), ("f32", 4, 2, 5), ("bf16", 32, 8, 40)])
def test_sparse_attention_reports_chunks_beyond_max_q_len(gpu, dt, H, kv, rows):
    # the rows up to the bound are computed, those beyond it left as they were
    rng = np.random.default_rng(13)
    bs, hd, top = 16, 64, 16
    cu = np.array([0, 1, 1 + rows])
    ctx = np.array([300, 400])
    tables, nb, _ = place(rng, ctx, bs)
    k, v = (rounded(rng.normal(size=(nb, bs, kv, hd)), dt) for _ in range(2))
    cache, pool = to_pool(dt, k, v, bs)
    q = rounded(rng.normal(size=(1 + rows, H, hd)), dt)
    blocks = choose(rng, ref.rows_of(cu, ctx), kv, top, bs, "select")
    want, bound = ref.sparse_attention(q, k, v, blocks, tables, cu, ctx, bs, hd ** -0.5)
    out = torch.full((1 + rows, H * hd), 5.0, dtype=torch.float32, device=gpu)
    pool.sparse_attention(torch.tensor(q).to(TD[dt]).to(gpu), i32(blocks, gpu), tables, ctx,
                          cu_q_lens=i32(cu, gpu), max_q_len=rows - 1, out=out)
    with pytest.raises(pagedkv.PagedKvError, match="length"):
        cache.check()
    got = out.double().cpu().numpy().reshape(q.shape)
    within(got[:-1], want[:-1], bound[:-1], "f32")
    assert (got[-1] == 5.0).all()
    out.fill_(5.0)
    got = run_sparse(gpu, dt, cache, pool, q, blocks, tables, cu, ctx, max_q_len=rows, out=out)
    within(got, want, bound, "f32")
    cache.close()


def test_sparse_attention_of_a_negative_context(gpu):
    # no keys: a zero row, and nothing to report while its list is empty
    cache = pagedkv.PagedKvCache(1, 10, 16, 2, 64, torch.bfloat16)
    q = torch.ones((3, 4, 64), dtype=torch.bfloat16, device=gpu)
    blocks = torch.full((3, 2, 4), -1, dtype=torch.int32, device=gpu)
    tables = torch.zeros((3, 8), dtype=torch.int32, device=gpu)
    out = cache.layer(0).sparse_attention(q, blocks, tables, i32([-40, 0, -2 ** 31], gpu))
    cache.check()
    assert (out == 0).all()
    cache.close()


def test_sparse_attention_of_a_ragged_batch_without_max_q_len(gpu):
    # 1024 requests, 4224 rows, 16 heads: as a launch of 4224 rows a request this is
    # 4.3 million (row, kv head) items; no part is joined, so heads do not count
    rng = np.random.default_rng(14)
    bs, kv, hd, H, n = 16, 1, 64, 16, 1024
    m = np.ones(n, np.int64)
    m[0] = 3201
    cu = np.concatenate(([0], np.cumsum(m)))
    ctx = np.full(n, 60)
    ctx[0] = 3201
    cache = pagedkv.PagedKvCache(1, 300, bs, kv, hd, torch.bfloat16)
    pool = cache.layer(0)
    slots = torch.arange(300 * bs, dtype=torch.int32, device=gpu)
    k, v = (torch.tensor(rng.normal(size=(300 * bs, kv, hd))).bfloat16().to(gpu) for _ in range(2))
    pool.append(k, v, slots)
    tables = i32(rng.integers(0, 300, (n, 201)), gpu)
    rows = ref.rows_of(cu, ctx)
    blocks = i32(choose(rng, rows, kv, 4, bs, "select"), gpu)
    q = torch.tensor(rng.normal(size=(len(rows), H, hd))).bfloat16().to(gpu)
    args = (q, blocks, tables, i32(ctx, gpu), i32(cu, gpu))
    got = pool.sparse_attention(*args)
    want = pool.sparse_attention(*args, max_q_len=3201)
    cache.check()
    assert torch.equal(got, want)
    cache.close()


@pytest.mark.parametrize("on_host", [list, np.asarray, torch.tensor])
def test_bound_of_chunks_on_the_host_is_the_longest(gpu, on_host):
    # 4096 requests, one of two rows: all rows as the bound of each would be refused
    rng = np.random.default_rng(15)
    bs, kv, hd, H, n = 16, 4, 64, 4, 4096
    m = np.ones(n, np.int64)
    m[7], m[9] = 2, 0
    cu = np.concatenate(([0], np.cumsum(m)))
    ctx = rng.integers(2, 200, n)
    cache, pool = to_pool("bf16", *rng.normal(size=(2, 50, bs, kv, hd)), bs)
    tables = i32(rng.integers(0, 50, (n, 13)), gpu)
    bounds = pool.update_key_bounds(pool.new_key_bounds(), i32(np.arange(50)[None], gpu),
                                    i32([50 * bs], gpu))
    q = torch.tensor(rng.normal(size=(cu[-1], H, hd))).bfloat16().to(gpu)
    args, given = (tables, i32(ctx, gpu)), dict(cu_q_lens=i32(cu, gpu), max_q_len=2)
    cu = on_host(cu.tolist())
    want = pool.select_blocks(q, bounds, *args, 5, 1, 2, **given)
    assert torch.equal(pool.select_blocks(q, bounds, *args, 5, 1, 2, cu_q_lens=cu), want)
    assert torch.equal(pool.sparse_attention(q, want, *args, cu_q_lens=cu),
                       pool.sparse_attention(q, want, *args, **given))
    cache.check()
    cache.close()


def test_offsets_past_32_bits(gpu):
    # 2.1 million slots of 2 KiB rows: the last blocks lie beyond 4 GiB
    bs, kv, hd, nb = 256, 8, 128, 9000
    rng = np.random.default_rng(10)
    cache = pagedkv.PagedKvCache(1, nb, bs, kv, hd, torch.bfloat16)
    pool = cache.layer(0)
    ctx = np.array([700, 300])
    tables = np.array([[nb - 1, 4, nb - 5], [nb - 7, nb - 2, 0]])
    kr, vr = (rounded(rng.normal(size=(2, 3 * bs, kv, hd)), "bf16") for _ in range(2))
    small_k, small_v = (np.zeros((6, bs, kv, hd)) for _ in range(2))
    for s in range(2):
        slots = (tables[s][:, None] * bs + np.arange(bs)).reshape(-1)
        pool.append(*(torch.tensor(x[s]).bfloat16().to(gpu) for x in (kr, vr)), slots.astype(np.int32))
        small_k[3 * s:3 * s + 3] = kr[s].reshape(3, bs, kv, hd)
        small_v[3 * s:3 * s + 3] = vr[s].reshape(3, bs, kv, hd)
    st = np.array([[0, 1, 2], [3, 4, 5]])
    q = rounded(rng.normal(size=(2, 16, hd)), "bf16")
    blocks = np.tile([0, 2, -1], (2, kv, 1))
    blocks[1] = [0, 1, -1]
    want, bound = ref.sparse_attention(q, small_k, small_v, blocks, st, None, ctx, bs, hd ** -0.5)
    got = run_sparse(gpu, "bf16", cache, pool, q, blocks, tables, None, ctx, out_dtype=torch.float32)
    within(got, want, bound, "f32")
    bounds = pool.update_key_bounds(pool.new_key_bounds(), tables, ctx)
    cache.check()
    wb = ref.key_bounds(np.zeros((6, kv, 2, hd)), small_k, st, np.zeros(2, int), ctx, bs)
    assert np.array_equal(bounds[torch.tensor(tables.reshape(-1))[[0, 1, 2, 3, 4]]].double().cpu().numpy(),
                          wb[[0, 1, 2, 3, 4]])
    cache.close()


# ---------------------------------------------------------------------------
# draft verification
# ---------------------------------------------------------------------------
def verify_case(seed, batch, vocab, k, dt, ddt, sharp=3.0):
    rng = np.random.default_rng(seed)
    n = rng.integers(0, k + 1, batch)
    cu = np.concatenate(([0], np.cumsum(n)))
    rows, total = cu[-1] + batch, cu[-1]
    x = rounded(rng.normal(size=(rows, vocab)) * sharp, dt)
    temps = np.where(rng.random(batch) < 0.2, 0.0, rng.random(batch) + 0.3).astype(np.float32)
    y = np.zeros((total, vocab))
    d = np.zeros(total, np.int64)
    for b in range(batch):
        for i in range(n[b]):
            y[cu[b] + i] = rounded(x[cu[b] + b + i] + rng.normal(size=vocab) * 0.5, ddt)
            if temps[b] == 0 or vocab == 1:
                d[cu[b] + i] = np.argmax(y[cu[b] + i])
            else:
                w = np.exp((y[cu[b] + i] - y[cu[b] + i].max()) / temps[b])
                d[cu[b] + i] = rng.choice(vocab, p=w / w.sum())
    u = rng.random(total).astype(np.float32)
    ul = rng.random(batch).astype(np.float32)
    return x, d, cu, u, ul, y, temps


def run_verify(gpu, dt, ddt, x, d, cu, u, ul, y, temps, stride=0, **kw):
    def rows(a, t):
        a = torch.tensor(a).to(TD[t]).to(gpu)
        if not stride or not a.numel():
            return a
        wide = torch.full((a.shape[0], a.shape[1] + stride), 99.0, dtype=a.dtype, device=gpu)
        wide[:, :a.shape[1]] = a
        return wide[:, :a.shape[1]]

    tok, acc = pagedkv.verify_drafts(
        rows(x, dt), i32(d, gpu), i32(cu, gpu), torch.tensor(u).to(gpu), torch.tensor(ul).to(gpu),
        draft_logits=None if y is None else rows(y, ddt),
        temperatures=None if temps is None else torch.tensor(temps).to(gpu), **kw)
    torch.cuda.synchronize()
    return host(tok), host(acc)


def same_verify(got, want):
    assert np.array_equal(got[1], want[1])
    assert np.array_equal(got[0], want[0])


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("dt,ddt,batch,vocab,k,stride", [
    ("bf16", "bf16", 5, 1000, 4, 0), ("f32", "f32", 3, 5001, 5, 0), ("f16", "f32", 9, 77, 3, 3),
    ("bf16", "f16", 1, 40000, 8, 8), ("f32", "bf16", 70, 33, 6, 1), ("f16", "f16", 4, 1, 3, 0),
    ("bf16", "f32", 2, 2, 2, 0), ("f32", "f32", 2, 20000, 300, 4), ("bf16", "bf16", 300, 130, 2, 6),
    ("f16", "bf16", 1, 9000, 1, 0), ("bf16", "bf16", 4500, 12, 2, 0), ("f32", "f32", 65, 40, 1, 0)])
def test_verify(gpu, dt, ddt, batch, vocab, k, stride, draft):
    a = verify_case(batch * 31 + vocab, batch, vocab, k, dt, ddt)
    x, d, cu, u, ul, y, temps = a
    y = y if draft else None
    want = ref.verify(x, d, cu, u, ul, y, temps)
    same_verify(run_verify(gpu, dt, ddt, x, d, cu, u, ul, y, temps, stride), want)


def test_verify_greedy_without_temperatures(gpu):
    x, d, cu, u, ul, y, _ = verify_case(3, 20, 300, 5, "bf16", "bf16")
    x = np.round(x)  # equal maxima: the first one counts
    for r, t in enumerate(d):
        if r % 3:
            d[r] = np.argmax(x[r + np.searchsorted(cu[1:], r, side="right")])
    want = ref.verify(x, d, cu, u, ul, y, None)
    assert 0 < want[1].sum() < len(d)
    same_verify(run_verify(gpu, "bf16", "bf16", x, d, cu, u, ul, y, None), want)
    same_verify(run_verify(gpu, "bf16", "bf16", x, d, cu, u, ul, None, None), want)
    same_verify(run_verify(gpu, "bf16", "bf16", x, d, cu, u, ul, y, np.zeros(20, np.float32)), want)


@pytest.mark.parametrize("dt,draft", [("bf16", False), ("bf16", True), ("f32", False)])
def test_verify_draws_at_a_boundary(gpu, dt, draft):
    # numbers that put the running sum 2e-11 to 1e-9 beside a token's end: more than
    # sums in 64 bits are off by (relative to their total, vocab 2^-53 < 1.5e-11 and the
    # weights' own 1e-14), far less than 32-bit exponentials are
    rng = np.random.default_rng(17)
    vocab, batch = 128256, 48
    x = rounded(rng.normal(size=vocab) * 2, dt)
    y = rounded(x + rng.normal(size=vocab) * 0.7, dt)
    w = np.exp(x.astype(np.float64) - x.max())
    w /= w.sum()
    tok = int(np.argmax(y - x))  # q above p: not kept by a number near 1
    if draft:
        q = np.exp(y.astype(np.float64) - y.max())
        w = np.maximum(w - q / q.sum(), 0.0)
    ends = np.cumsum(w)
    ends /= ends[-1]
    near = ends.astype(np.float32)
    off = np.abs(near.astype(np.float64) - ends)
    at = np.flatnonzero((off > 2e-11) & (off < 1e-9) & (near > 0) & (near < 1) & (w > 0))
    at = rng.choice(at, batch, replace=False)
    n = int(draft)
    cu = np.arange(batch + 1) * n
    u = np.full(batch * n, 1 - 2.0 ** -24, np.float32)
    got = run_verify(gpu, dt, dt, np.tile(x, (batch * (n + 1), 1)), np.full(batch * n, tok), cu, u,
                     near[at], np.tile(y, (batch, 1)) if draft else None, np.ones(batch, np.float32))
    want = (ends > near[at].astype(np.float64)[:, None]).argmax(1)
    assert (got[1] == 0).all()
    assert np.array_equal(got[0].reshape(batch, n + 1)[:, 0], want)


@pytest.mark.parametrize("t", [-1.0, -0.0, np.nan, np.inf, -np.inf])
def test_verify_temperatures_that_are_greedy(gpu, t):
    # every third request has such a temperature; the others draw
    x, d, cu, u, ul, y, temps = verify_case(11, 21, 700, 4, "f32", "bf16")
    temps = np.maximum(temps, np.float32(0.3))
    zero, given = temps.copy(), temps.copy()
    zero[::3], given[::3] = 0.0, t
    want = ref.verify(x, d, cu, u, ul, y, zero)
    same_verify(run_verify(gpu, "f32", "bf16", x, d, cu, u, ul, y, given), want)


@pytest.mark.parametrize("what", ["masked", "empty", "nan", "inf", "tokens", "edges", "same", "flat",
                                  "cold", "emptydraft", "lowest", "huge", "offset"])
@pytest.mark.parametrize("draft", [True, False])
def test_verify_odd_values(gpu, what, draft):
    x, d, cu, u, ul, y, temps = verify_case(17, 24, 4700, 4, "f32", "f32")
    rng = np.random.default_rng(1)
    if what == "masked":  # a distribution cut to a few tokens
        x[rng.random(x.shape) < 0.999] = -np.inf
        y[rng.random(y.shape) < 0.99] = -np.inf
    elif what == "empty":
        x[::3] = -np.inf
    elif what == "emptydraft":
        y[::2] = -np.inf
    elif what == "nan":
        x[:, ::7] = np.nan
        y[:, 1::5] = np.nan
    elif what == "inf":
        x[1::4, 33] = np.inf
        x[1::4, 4000] = np.inf
        y[::3, 33] = np.inf
    elif what == "tokens":
        d[::4], d[1::4] = -1, 4700
        d[2::8] = 2 ** 31 - 1
    elif what == "edges":
        u[:], ul[:] = 0.0, np.float32(1) - np.float32(2.0 ** -24)
        ul[::2] = 0.0
    elif what == "same":  # p == q: everything is kept
        for b in range(24):
            y[cu[b]:cu[b + 1]] = x[cu[b] + b:cu[b + 1] + b]
    elif what == "flat":
        x[:], y[:] = 0.0, 1.0
    elif what == "lowest":  # masked by the type's lowest value, whole stretches of a row
        low = np.finfo(np.float32).min
        x[:, :3000], y[:, 200:] = low, low
        x[::2, 3500:], y[::3, :190] = low, low
    elif what == "huge":
        x *= 1e37
        y *= 1e30
    elif what == "offset":  # all of a row far from 0
        x += np.where(np.arange(len(x)) % 2, 1e9, -3e5)[:, None]
        y -= 1e7
        x, y = x.astype(np.float32).astype(np.float64), y.astype(np.float32).astype(np.float64)
    else:
        temps[:] = np.where(temps > 0, np.float32(0.01), 0)
    y = y if draft else None
    want = ref.verify(x, d, cu, u, ul, y, temps)
    same_verify(run_verify(gpu, "f32", "f32", x, d, cu, u, ul, y, temps), want)
    if what == "same" and draft:
        assert (want[1] == np.diff(cu))[temps > 0].all()


def masked_case(seed, dt, mask, temps, vocab=9000):
    """Requests of one to three live tokens a row, all others at `mask`; the live
    ones lie beyond the first tokens that a thread meets (2048) of a chunk."""
    rng = np.random.default_rng(seed)
    batch, k = 4 * len(temps), 2
    cu = np.arange(batch + 1) * k
    x, y = np.full((batch * (k + 1), vocab), mask), np.full((batch * k, vocab), mask)
    at = np.concatenate((np.arange(2050, 4300), np.arange(6700, 8900)))
    d = np.zeros(batch * k, np.int64)
    for r in range(len(x)):
        b, i = divmod(r, k + 1)
        live = rng.choice(at, 1 + r % 3, replace=False)
        x[r, live] = rng.normal(size=len(live)) * 2
        if i < k:
            y[b * k + i, live] = rng.normal(size=len(live)) * 2
            y[b * k + i, rng.choice(at)] = 1.0
            d[b * k + i] = rng.choice(live) if r % 5 else rng.choice(at)
    u, ul = (rng.random(n).astype(np.float32) for n in (batch * k, batch))
    return rounded(x, dt), d, cu, u, ul, rounded(y, dt), np.tile(np.float32(temps), 4)


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("dt,mask", [(t, m) for t in ("f32", "bf16") for m in (
    -1e4, -1e7, -2e7, -5e7, -8e7, -1e8, -1.2e8, -2e8, -3e8, -1e9)] + [("f16", -65504.0)])
def test_verify_logits_masked_by_a_finite_value(gpu, dt, mask, draft):
    temps = [1e-3, 3e-3, 0.01, 0.2, 0.3, 0.35, 0.5, 0.7, 0.8, 0.9, 1.0, 1.2]
    x, d, cu, u, ul, y, temps = masked_case(7, dt, mask, temps)
    y = y if draft else None
    want = ref.verify(x, d, cu, u, ul, y, temps)
    same_verify(run_verify(gpu, dt, dt, x, d, cu, u, ul, y, temps), want)


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_verify_temperatures_near_zero(gpu, dt, draft):
    x, d, cu, u, ul, y, temps = verify_case(29, 24, 9000, 4, dt, dt)
    x[1::2], y[1::2] = rounded(x[1::2] + 64, dt), rounded(y[1::2] + 10, dt)
    temps = np.tile(np.float32([1e-5, 1e-6, 4e-7, 1e-7, 3e-8, 1e-9]), 4)
    y = y if draft else None
    for r in range(0, len(d), 2):  # half of the drafts are the row's maximum
        d[r] = np.argmax(x[r + np.searchsorted(cu[1:], r, side="right")])
    want = ref.verify(x, d, cu, u, ul, y, temps)
    assert 0 < want[1].sum() < len(d)
    same_verify(run_verify(gpu, dt, dt, x, d, cu, u, ul, y, temps), want)


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("t", [2.5e35, 4e35, 1e37, 3e38])
def test_verify_enormous_temperatures(gpu, t, draft):
    # every token that is not at -inf is as likely, the others have probability 0
    x, d, cu, u, ul, y, _ = verify_case(31, 24, 4700, 4, "f32", "f32")
    rng = np.random.default_rng(2)
    x[rng.random(x.shape) < 0.6] = -np.inf
    y[rng.random(y.shape) < 0.4] = -np.inf
    x[::4, 100] = 1e38
    x[1::4, 5:2000] = -np.finfo(np.float32).max
    y[::3, 7] = -3e38
    y = y if draft else None
    temps = np.full(24, t, np.float32)
    want = ref.verify(x, d, cu, u, ul, y, temps)
    same_verify(run_verify(gpu, "f32", "f32", x, d, cu, u, ul, y, temps), want)


def test_verify_without_any_draft(gpu):
    x, d, cu, u, ul, y, temps = verify_case(23, 6, 500, 0, "bf16", "bf16")
    want = ref.verify(x, d, cu, u, ul, None, temps)
    same_verify(run_verify(gpu, "bf16", "bf16", x, d, cu, u, ul, None, temps), want)
    same_verify(run_verify(gpu, "bf16", "bf16", x, d, cu, u, ul, y, temps), want)


# ---------------------------------------------------------------------------
# together: a toy model's speculative steps, lengths never leaving the device
# ---------------------------------------------------------------------------
class Toy:
    """One attention layer over a paged pool, two embeddings and a readout; its
    draft model is the readout of the token alone."""

    def __init__(self, gpu, seed=0, vocab=97, H=4, kv=2, hd=64):
        g = torch.Generator(device="cpu").manual_seed(seed)
        r = lambda *s: torch.randn(s, generator=g).to(gpu)  # noqa: E731
        self.V, self.H, self.kv, self.hd = vocab, H, kv, hd
        self.eq, self.ek, self.ev = r(vocab, H, hd), r(vocab, kv, hd), r(vocab, kv, hd)
        self.out, self.skip = r(H * hd, vocab) * 0.3, r(vocab, vocab) * 1.5

    def draft(self, tok):
        return self.skip[tok]

    def rows(self, tok):
        return tuple(e[tok].to(torch.bfloat16).contiguous() for e in (self.eq, self.ek, self.ev))

    def logits(self, attn, tok):
        return attn.float() @ self.out + self.skip[tok]


def spec_steps(gpu, toy, steps, k=3, n=5, bs=16, width=24, top=6, use_stream=None, seed=1):
    """Runs `steps` speculative steps; yields what each wrote, for the check."""
    rng = np.random.default_rng(seed)
    nb = n * width
    cache = pagedkv.PagedKvCache(1, nb, bs, toy.kv, toy.hd, torch.bfloat16)
    pool = cache.layer(0)
    bounds = pool.new_key_bounds()
    prompts = [rng.integers(0, toy.V, m) for m in (150, 3, 97, 200, 16)][:n]
    seq = i32(np.zeros(n), gpu)
    tables = torch.zeros((n, width), dtype=torch.int32, device=gpu)
    have, free = i32(np.zeros(n), gpu), i32(rng.permutation(nb), gpu)
    count = i32([nb], gpu)
    hist = [list(p) for p in prompts]
    # prompts: stored whole, all blocks' bounds
    lens = np.array([len(p) - 1 for p in prompts])  # the last token is fed with the drafts
    st = pagedkv.step_tables(seq, i32(lens, gpu), tables, have, free, count, bs, nb, int(lens.sum()))
    toks = torch.tensor(np.concatenate([p[:-1] for p in prompts]), device=gpu)
    _, kk, vv = toy.rows(toks)
    pool.append(kk, vv, st.slot_mapping)
    pool.update_key_bounds(bounds, st.block_tables, st.context_lens)
    seq, tables, have, count = st.context_lens, st.block_tables, st.n_blocks, st.free_count
    cur = torch.tensor([p[-1] for p in prompts], device=gpu)
    temps = torch.tensor([0.8, 0.0, 1.0, 0.6, 1.2][:n], device=gpu)
    new = i32(np.full(n, k + 1), gpu)
    cu_d = i32(np.arange(n + 1) * k, gpu)
    for step in range(steps):
        u, ul, du = (torch.tensor(rng.random(m), dtype=torch.float32, device=gpu)
                     for m in (n * k, n, n * k))
        d, q, prev = [], [], cur
        for i in range(k):  # the draft model draws by the inverse of its distribution
            lg = toy.draft(prev)
            p = torch.softmax(lg / temps.clamp(min=0.05)[:, None], 1)
            prev = (p.cumsum(1) < du.view(n, k)[:, i:i + 1]).sum(1).clamp(max=toy.V - 1)
            d.append(prev)
            q.append(lg)
        drafts, dl = torch.stack(d, 1), torch.stack(q, 1).reshape(n * k, toy.V)
        fed = torch.cat((cur[:, None], drafts), 1).reshape(-1)
        st = pagedkv.step_tables(seq, new, tables, have, free, count, bs, nb, n * (k + 1))
        qq, kk, vv = toy.rows(fed)
        pool.append(kk, vv, st.slot_mapping)
        pool.update_key_bounds(bounds, st.block_tables, st.context_lens, seq, k + 1)
        args = dict(cu_q_lens=st.cu_q_lens, max_q_len=k + 1)
        sel = pool.select_blocks(qq, bounds, st.block_tables, st.context_lens, top, 1, 2,
                                 max_context_len=bs * width, **args)
        attn = pool.sparse_attention(qq, sel, st.block_tables, st.context_lens, **args)
        tg = toy.logits(attn, fed)
        tok, acc = pagedkv.verify_drafts(tg, drafts.reshape(-1).int(), cu_d, u, ul, dl, temps)
        yield dict(hist=[list(h) for h in hist], fed=fed, st=st, sel=sel, attn=attn, tg=tg, tok=tok,
                   acc=acc, drafts=drafts, dl=dl, u=u, ul=ul, temps=temps, qq=qq)
        seq = seq + acc + 1  # the fed token and its kept drafts stay
        tables, have, count = st.block_tables, st.n_blocks, st.free_count
        t = tok.view(n, k + 1)
        cur = t.gather(1, acc[:, None].long())[:, 0].long()
        for b in range(n):
            hist[b] += t[b, :int(acc[b]) + 1].tolist()
    cache.check()
    cache.close()


def test_speculative_steps(gpu):
    toy = Toy(gpu)
    bs, top, k, n = 16, 6, 3, 5
    ek, ev = (e.to(torch.bfloat16).double().cpu().numpy() for e in (toy.ek, toy.ev))
    kept = 0
    for r in spec_steps(gpu, toy, 6, k, n, bs, top=top):
        assert host(r["st"].status).tolist() == [0]
        ctx = host(r["st"].context_lens)
        cu = host(r["st"].cu_q_lens)
        fed = r["fed"].view(n, k + 1).cpu().numpy()
        # contiguous copies of what the pool must hold: history, then the fed tokens
        nbk = max(-(-int(c) // bs) for c in ctx)
        K, V = (np.zeros((n * nbk, bs, 2, 64)) for _ in range(2))
        for b in range(n):
            toks = r["hist"][b][:-1] + fed[b].tolist()
            assert len(toks) == ctx[b]
            for j, t in enumerate(toks):
                K[b * nbk + j // bs, j % bs], V[b * nbk + j // bs, j % bs] = ek[t], ev[t]
        tab = np.arange(n * nbk).reshape(n, nbk)
        bounds = ref.key_bounds(np.zeros((n * nbk, 2, 2, 64)), K, tab, [0] * n, ctx, bs)
        q = r["qq"].double().cpu().numpy()
        sel = ref.select(q, bounds, tab, cu, ctx, bs, top, 1, 2)
        assert np.array_equal(host(r["sel"]), sel)
        want, bound = ref.sparse_attention(q, K, V, sel, tab, cu, ctx, bs, 0.125)
        within(r["attn"].double().cpu().numpy().reshape(want.shape), want, bound, "bf16")
        got = host(r["tok"]), host(r["acc"])
        same_verify(got, ref.verify(r["tg"].cpu().numpy(), host(r["drafts"].reshape(-1)),
                                    list(range(0, n * k + 1, k)), r["u"].cpu().numpy(),
                                    r["ul"].cpu().numpy(), r["dl"].cpu().numpy(),
                                    r["temps"].cpu().numpy()))
        kept += int(got[1].sum())
    assert kept > 0


def spec_operands(gpu, seed=5, n=6, k=2, H=8, kv=2, hd=64, bs=16, width=40, vocab=700):
    rng = np.random.default_rng(seed)
    ctx = rng.integers(100, width * bs - 10, n)
    tables, nb, free = place(rng, ctx, bs, spare=40, width=width)
    kk, vv = (rounded(rng.normal(size=(nb, bs, kv, hd)), "bf16") for _ in range(2))
    cache, pool = to_pool("bf16", kk, vv, bs)
    m = k + 1
    t = {"seq": i32(ctx - 1, gpu), "new": i32(np.full(n, m), gpu), "tables": i32(tables, gpu),
         "have": i32(-(-ctx // bs), gpu), "free": i32(free, gpu), "count": i32([len(free)], gpu),
         "q": torch.tensor(rng.normal(size=(n * m, H, hd))).bfloat16().to(gpu),
         "k": torch.tensor(rng.normal(size=(n * m, kv, hd))).bfloat16().to(gpu),
         "lg": torch.tensor(rng.normal(size=(n * m, vocab)) * 3).float().to(gpu),
         "dl": torch.tensor(rng.normal(size=(n * k, vocab)) * 3).float().to(gpu),
         "d": i32(rng.integers(0, vocab, n * k), gpu), "cu": i32(np.arange(n + 1) * k, gpu),
         "u": torch.tensor(rng.random(n * k)).float().to(gpu) * 0.2,
         "ul": torch.tensor(rng.random(n)).float().to(gpu),
         "tp": torch.tensor([0.7, 0.0, 1.0, 0.9, 2.0, 0.5][:n]).to(gpu)}
    bounds = pool.update_key_bounds(pool.new_key_bounds(), t["tables"], i32(ctx, gpu))

    def go(stream=None):
        st = pagedkv.step_tables(t["seq"], t["new"], t["tables"], t["have"], t["free"], t["count"],
                                 bs, nb, n * m, stream=stream)
        kw = dict(cu_q_lens=st.cu_q_lens, max_q_len=m, stream=stream)
        pool.append(t["k"], t["k"], st.slot_mapping, stream)
        pool.update_key_bounds(bounds, st.block_tables, st.context_lens, t["seq"], m, stream=stream)
        sel = pool.select_blocks(t["q"], bounds, st.block_tables, st.context_lens, 7, 1, 2, **kw)
        at = pool.sparse_attention(t["q"], sel, st.block_tables, st.context_lens, **kw)
        tok, acc = pagedkv.verify_drafts(t["lg"], t["d"], t["cu"], t["u"], t["ul"], t["dl"], t["tp"],
                                         stream=stream)
        return [*st, bounds, sel, at, tok, acc]

    return cache, t, go


def test_on_another_stream(gpu):
    cache, t, go = spec_operands(gpu)
    want = [x.clone() for x in go()]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    got = go(s)
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    cache.check()
    cache.close()


def test_captured_and_replayed(gpu):
    cache, t, go = spec_operands(gpu)
    go()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs of the same work, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = go()
        graphs.append((g, out))
    rng = np.random.default_rng(0)
    for i in range(4):
        t["q"].copy_(torch.tensor(rng.normal(size=t["q"].shape)).bfloat16())
        t["lg"].copy_(torch.tensor(rng.normal(size=t["lg"].shape) * 3))
        t["ul"].copy_(torch.tensor(rng.random(t["ul"].shape)))
        t["seq"].copy_(t["seq"] - i % 2)
        want = [x.clone() for x in go()]
        torch.cuda.synchronize()
        g, out = graphs[i % 2]
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)
    cache.check()
    cache.close()
    # (the graphs' memory goes with them)
    del graphs


def test_same_bits_on_every_run(gpu):
    cache, t, go = spec_operands(gpu, seed=6)
    want = [x.clone() for x in go()]
    for _ in range(5):
        for a, b in zip(go(), want):
            assert torch.equal(a, b)
    cache.close()


# ---------------------------------------------------------------------------
# refusals of the calls that need a pool: before anything is enqueued
# ---------------------------------------------------------------------------
@pytest.fixture(scope="module")
def small(gpu):
    cache = pagedkv.PagedKvCache(1, 10, 16, 2, 64, torch.bfloat16)
    z = torch.zeros((3, 4), dtype=torch.int32, device=gpu)
    yield cache, cache.layer(0), torch.zeros((3, 4, 64), dtype=torch.bfloat16, device=gpu), z, z[:, 0].contiguous()
    cache.close()


def test_select_refuses(small):
    cache, pool, q, bt, cl = small
    b = pool.new_key_bounds()
    for kw in (dict(top_blocks=0), dict(top_blocks=2, first_blocks=2), dict(top_blocks=5, last_blocks=0),
               dict(top_blocks=5, first_blocks=-1), dict(top_blocks=5, max_context_len=0),
               dict(top_blocks=5, max_context_len=(1 << 30) + 1), dict(top_blocks=5, max_q_len=2),
               dict(top_blocks=1 << 28)):
        with pytest.raises(pagedkv.PagedKvError):
            pool.select_blocks(q, b, bt, cl, **kw, out=torch.empty(
                (3, 2, kw["top_blocks"]), dtype=torch.int32, device=q.device)
                if kw["top_blocks"] < 100 else None)
    for bad in (q[:2], q[:, :, :32].contiguous()):
        with pytest.raises(ValueError):
            pool.select_blocks(bad, b, bt, cl, 4)
    with pytest.raises(TypeError):
        pool.select_blocks(q.float(), b, bt, cl, 4)
    with pytest.raises(pagedkv.PagedKvError):  # three heads over two kv heads
        pool.select_blocks(q[:, :3].contiguous(), b, bt, cl, 4)
    for bad in (b[:5], b.cpu(), b.transpose(1, 2)):
        with pytest.raises(ValueError):
            pool.select_blocks(q, bad, bt, cl, 4)


def test_sparse_attention_refuses(small):
    cache, pool, q, bt, cl = small
    bl = torch.zeros((3, 2, 4), dtype=torch.int32, device=q.device)
    for kw in (dict(scale=float("nan")), dict(max_q_len=2), dict(out_dtype=torch.float16)):
        with pytest.raises(pagedkv.PagedKvError):
            pool.sparse_attention(q, bl, bt, cl, **kw)
    with pytest.raises(pagedkv.PagedKvError):
        pool.sparse_attention(q, bl[:, :, :0].contiguous(), bt, cl)
    for args in ((q, bl[:, :1], bt, cl), (q, bl, bt[:2], cl), (q, bl.cpu(), bt, cl)):
        with pytest.raises(ValueError):
            pool.sparse_attention(*args)
    with pytest.raises(TypeError):
        pool.sparse_attention(q, bl.long(), bt, cl)
    with pytest.raises(ValueError):
        pool.sparse_attention(q, bl, bt, cl, out=torch.empty((3, 100), device=q.device))
    L = pagedkv.lib()
    need = L.pkv_sparse_workspace_bytes(cache.handle, 3, 4, 400)
    assert need > 0
    out = torch.zeros((3, 256), device=q.device)
    rc = L.pkv_sparse_attention(cache.handle, 0, q.data_ptr(), out.data_ptr(), pagedkv.F32,
                                bl.data_ptr(), 400, None, cl.data_ptr(), bt.data_ptr(), 4, 3, 3, 1, 4,
                                0.1, out.data_ptr(), need - 1, None)
    assert rc == pagedkv._lib.PKV_ERR_INVALID and b"workspace" in L.pkv_last_error(cache.handle)


def test_key_bounds_refuses(small):
    cache, pool, q, bt, cl = small
    b = pool.new_key_bounds()
    for n in (0, -1, (1 << 30) + 1):
        with pytest.raises(pagedkv.PagedKvError):
            pool.update_key_bounds(b, bt, cl, max_new_len=n)
    with pytest.raises(ValueError):
        pool.update_key_bounds(b, bt[:1], cl)
    with pytest.raises(ValueError):
        pool.update_key_bounds(b[:, :1], bt, cl)
    with pytest.raises(TypeError):
        pool.update_key_bounds(b.float(), bt, cl)


def test_empty_batches(small):
    cache, pool, q, bt, cl = small
    b = pool.new_key_bounds()
    assert pool.select_blocks(q[:0], b, bt[:0], cl[:0], 4).shape == (0, 2, 4)
    assert pool.sparse_attention(q[:0], torch.zeros((0, 2, 4), dtype=torch.int32, device=q.device),
                                 bt[:0], cl[:0]).shape == (0, 256)
    pool.update_key_bounds(b, bt[:0], cl[:0])
    cache.check()
