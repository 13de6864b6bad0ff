"""Serving from a cache held in 4 bits on the GPU: rows into the pool and back,
attention over it, packed prompt attention and adjusted logits, each against its
plain 64-bit implementation (serve4_ref), then together."""
import math

import numpy as np
import pytest
import torch

import pagedkv
import serve4_ref as ref

pytestmark = pytest.mark.gpu

TD = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step
# what a weight is rounded by before it meets a value: attention over 4 bits takes two
# f16, prompt attention the type of its inputs
Q4_WEIGHT = 2.0 ** -21
PROMPT_WEIGHT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def i32(x, gpu):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=gpu)


def typed(x, dt, gpu):
    """x rounded to the type: (device tensor, float64 values)."""
    t = torch.tensor(np.asarray(x)).to(TD[dt])
    return t.to(gpu), t.double().numpy()


def host(t):
    return t.double().cpu().numpy()


def keys_values(rng, n, kv, hd):
    k = rng.normal(size=(n, kv, hd)) + rng.normal(size=(kv, hd)) * rng.choice([0.5, 5.0], (kv, hd))
    return k, rng.normal(size=(n, kv, hd))


# ---------------------------------------------------------------------------
# rows into the pool and back
# ---------------------------------------------------------------------------
def special_rows(rng, n, kv, hd):
    """Rows with groups that are constant, zero, tiny, huge, not finite, or on borders."""
    x = rng.normal(size=(n, kv, hd))
    g = x.reshape(n * kv, hd // 32, 32)
    kinds = rng.integers(0, 10, g.shape[:2])
    for (r, j), kind in np.ndenumerate(kinds):
        if kind == 0:
            g[r, j] = 0.25
        elif kind == 1:
            g[r, j] = 0.0
        elif kind == 2:
            g[r, j] *= 1e-7
        elif kind == 3:
            g[r, j] *= 3e4
        elif kind == 4:
            g[r, j, :3] = (np.nan, np.inf, -np.inf)
        elif kind == 5:  # steps of exactly 1, elements halfway between codes
            g[r, j] = rng.integers(0, 30, 32) * 0.5
            g[r, j, :2] = (0.0, 15.0)
        elif kind == 6:
            g[r, j] += 1000.0
    return x


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd,kv,bs", [(64, 3, 16), (128, 2, 32), (256, 1, 64), (128, 5, 256)])
def test_append_holds_the_codes_and_gather_gives_their_values(gpu, dt, hd, kv, bs):
    rng = np.random.default_rng(hd + kv)
    n, nb = 75, 7
    k, kx = typed(special_rows(rng, n, kv, hd), dt, gpu)
    v, vx = typed(special_rows(rng, n, kv, hd), dt, gpu)
    slots = rng.permutation(nb * bs)[:n]
    slots[5] = -1
    cache = pagedkv.PagedKvCache(2, nb, bs, kv, hd, pagedkv.Q4)
    assert cache.layer_bytes == nb * bs * kv * hd * 5 // 8
    pool = cache.layer(1)
    pool.q4_append(k, v, i32(slots, gpu))
    cache.check()
    written = np.delete(np.arange(n), 5)
    for which, x in ((pagedkv.K, kx), (pagedkv.V, vx)):
        c, m, s = ref.quantize(x)
        codes = np.zeros((nb * bs, kv, hd), np.int64)
        ms, ss = np.zeros((2, nb * bs, kv, hd // 32))
        codes[slots[written]], ms[slots[written]], ss[slots[written]] = c[written], m[written], s[written]
        got = cache.read_bytes(1, which).reshape(nb, kv, -1)
        for b in range(nb):
            for h in range(kv):
                rows = slice(b * bs, (b + 1) * bs)
                want = ref.chunk_bytes(which == pagedkv.K, codes[rows, h], ms[rows, h], ss[rows, h],
                                       bs)
                assert np.array_equal(got[b, h], want), (which, b, h)
        assert not cache.read_bytes(0, which).any()
    # values back: m + s c is exact in 64 bits, rounded to f32 and then to the type
    for odt in ("f32", "f16", "bf16"):
        out = pool.q4_gather(i32(slots, gpu), out_dtype=TD[odt])
        for o, x in zip(out, (kx, vx)):
            want = ref.held(x)
            want[5] = 0.0
            assert torch.equal(o.cpu(), torch.tensor(want).float().to(TD[odt]))
    cache.check()


def test_append_reads_rows_at_a_stride(gpu):
    rng = np.random.default_rng(3)
    n, kv, hd, bs = 37, 4, 64, 16
    x, xx = typed(rng.normal(size=(n, 3 * kv, hd)), "bf16", gpu)
    cache = pagedkv.PagedKvCache(1, 4, bs, kv, hd, pagedkv.Q4)
    pool, slots = cache.layer(0), i32(np.arange(n), gpu)
    pool.q4_append(x[:, kv:2 * kv], x[:, 2 * kv:], slots)
    for o, want in zip(pool.q4_gather(slots), (xx[:, kv:2 * kv], xx[:, 2 * kv:])):
        assert np.array_equal(host(o), ref.held(want).astype(np.float32))
    # heads apart, or the channels: copied first
    y = x.transpose(0, 1).contiguous().transpose(0, 1)
    pool.q4_append(y[:, :kv], y[:, kv:2 * kv], slots)
    assert np.array_equal(host(pool.q4_gather(slots)[0]), ref.held(xx[:, :kv]).astype(np.float32))


def test_slots_beyond_the_pool_are_reported(gpu):
    cache = pagedkv.PagedKvCache(1, 2, 16, 2, 64, pagedkv.Q4)
    pool = cache.layer(0)
    x = torch.ones((3, 2, 64), device=gpu)
    pool.q4_append(x, x, i32([1, 32, 2 ** 31 - 1], gpu))
    with pytest.raises(pagedkv.PagedKvError, match="slot-out-of-range"):
        cache.check()
    k, v = pool.q4_gather(i32([1, 32, -5], gpu))
    with pytest.raises(pagedkv.PagedKvError, match="slot-out-of-range"):
        cache.check()
    assert torch.all(k[0] == 1) and not k[1:].any() and not v[1:].any()
    got = cache.read_bytes(0, pagedkv.K)
    pool.q4_append(x, x, i32([-1, -1, -7], gpu))
    pool.q4_append(x[:0], x[:0], i32([], gpu))
    assert np.array_equal(got, cache.read_bytes(0, pagedkv.K))
    cache.check()


def test_blocks_are_copied_and_compacted(gpu):
    rng = np.random.default_rng(4)
    kv, hd, bs, nb = 2, 128, 16, 9
    k, kx = typed(rng.normal(size=(nb * bs, kv, hd)), "f16", gpu)
    cache = pagedkv.PagedKvCache(2, nb, bs, kv, hd, pagedkv.Q4)
    slots = torch.arange(nb * bs, dtype=torch.int32, device=gpu)
    for layer in range(2):
        cache.layer(layer).q4_append(k, -k, slots)
    want = ref.held(kx).reshape(nb, bs, kv, hd)
    cache.copy_blocks([0, 3], [8, 7])
    want[[8, 7]] = want[[0, 3]]
    cache.compact([8, 2, 5], [2, 5, 0])
    want[[2, 5, 0]] = want[[8, 2, 5]]
    cache.check()
    for layer in range(2):
        for b in (0, 2, 5, 7, 1, 3):
            got = cache.layer(layer).q4_gather(slots[b * bs:(b + 1) * bs])[0]
            assert np.array_equal(host(got), want[b].astype(np.float32))


def test_rows_past_32_bit_offsets(gpu):
    # a layer's K of 6 GB: slots on both sides of 2^32 bytes, stored, read and attended
    kv, hd, bs = 8, 128, 16
    nb = 600_000
    cache = pagedkv.PagedKvCache(1, nb, bs, kv, hd, pagedkv.Q4)
    assert cache.layer_bytes > 1 << 32
    pool, rng = cache.layer(0), np.random.default_rng(5)
    k, v = keys_values(rng, 40, kv, hd)
    k, kx = typed(k, "bf16", gpu)
    v, vx = typed(v, "bf16", gpu)
    blocks = np.array([nb - 1, 5, nb // 2 + 3])
    slots = (blocks[:, None] * bs + np.arange(bs)).reshape(-1)[:40]
    pool.q4_append(k, v, i32(slots, gpu))
    assert np.array_equal(host(pool.q4_gather(i32(slots, gpu))[1]), ref.held(vx).astype(np.float32))
    q, qx = typed(rng.normal(size=(1, 32, hd)), "bf16", gpu)
    o = pool.q4_attention(q, i32(blocks[None], gpu), i32([40], gpu))
    cache.check()
    want, *abc = ref.attention(qx, ref.held(kx), ref.held(vx), 1, hd ** -0.5, ref.held_terms(kx),
                               ref.held_terms(vx))
    tol = ref.tolerance(want, *abc, 40, hd, Q4_WEIGHT, HALF["bf16"])
    assert np.all(np.abs(host(o).reshape(want.shape) - want) <= tol)
    cache.close()


# ---------------------------------------------------------------------------
# attention over the pool
# ---------------------------------------------------------------------------
class Case:
    """Sequences in a pool of 4 bits, their rows' queries, and the plain result."""

    def __init__(self, gpu, seed, dt, h, kv, hd, bs, ctx, q_lens=None, scale=None, k_by=1.0,
                 v_by=1.0, q_by=1.0, spare=3):
        rng = np.random.default_rng(seed)
        self.rng, self.gpu, self.dt, self.h, self.hd = rng, gpu, dt, h, hd
        self.scale = hd ** -0.5 if scale is None else scale
        need = [-(-c // bs) for c in ctx]
        nb = sum(need) + spare
        perm = rng.permutation(nb)
        self.tables = np.full((len(ctx), max(max(need), 1)), nb + 5)  # never read
        at = 0
        for i, n in enumerate(need):
            self.tables[i, :n] = perm[at:at + n]
            at += n
        k, v = keys_values(rng, nb * bs, kv, hd)
        k, self.k = typed(k * k_by, dt, gpu)
        v, self.v = typed(v * v_by, dt, gpu)
        self.take(self.k, self.v)
        self.cache = pagedkv.PagedKvCache(1, nb, bs, kv, hd, pagedkv.Q4)
        self.pool = self.cache.layer(0)
        self.pool.q4_append(k, v, torch.arange(nb * bs, dtype=torch.int32, device=gpu))
        self.q_lens = [1] * len(ctx) if q_lens is None else list(q_lens)
        self.cu = None if q_lens is None else np.concatenate(([0], np.cumsum(q_lens)))
        self.ctx, self.bs = list(ctx), bs
        self.q, self.qx = typed(rng.normal(size=(sum(self.q_lens), h, hd)) * q_by, dt, gpu)

    def take(self, k, v):
        """k, v have been stored in all slots."""
        self.k, self.v = ref.held(k), ref.held(v)
        self.terms = ref.held_terms(k), ref.held_terms(v)

    def rows(self, s):
        pos = np.arange(self.ctx[s])
        at = self.tables[s, pos // self.bs] * self.bs + pos % self.bs
        return (self.k[at], self.v[at]), [t[at] for t in self.terms]

    def steps(self, m):
        """What a chunk's weights, keys and values are rounded by.  Chunks of more
        than 32 columns (rows times heads of a kv head) of 16-bit queries take f16
        values, and for bf16 also keys and weights."""
        r, few = self.h // self.k.shape[1], 2 * 512 // self.hd
        if self.dt == "f32" or max(self.q_lens) * r <= 32 or (r <= few and m * r <= few):
            return dict(weight_step=Q4_WEIGHT)
        step = 2.0 ** -11
        if self.dt == "f16":
            return dict(weight_step=Q4_WEIGHT, value_step=step)
        return dict(weight_step=step, value_step=step, key_step=step)

    def run(self, **kw):
        cu = None if self.cu is None else i32(self.cu, self.gpu)
        kw.setdefault("max_q_len", max(self.q_lens))
        kw.setdefault("max_context_len", max(max(self.ctx), 1))
        kw.setdefault("scale", self.scale)
        return self.pool.q4_attention(self.q, i32(self.tables, self.gpu), i32(self.ctx, self.gpu),
                                      cu_q_lens=cu, **kw)

    def check(self, out, out_dt=None, skip=()):
        at = 0
        got = host(out).reshape(-1, self.h, self.hd)
        for s, m in enumerate(self.q_lens):
            if s not in skip and m:
                kv, terms = self.rows(s)
                want, *abc = ref.attention(self.qx[at:at + m], *kv, m, self.scale, *terms)
                tol = ref.tolerance(want, *abc, self.ctx[s], self.hd, **self.steps(m),
                                    out_step=HALF[out_dt or self.dt])
                err = np.abs(got[at:at + m] - want)
                assert np.all(err <= tol), (s, m, self.ctx[s], float((err / tol).max()))
                assert not got[at:at + m][abc[0].sum(-1) == 0].any()  # rows without keys are zero
            at += m


SHAPES = [("bf16", 32, 8, 128), ("f16", 32, 8, 64), ("f32", 14, 2, 64), ("bf16", 64, 8, 128),
          ("f16", 8, 8, 128), ("bf16", 16, 8, 256), ("f32", 32, 4, 128), ("f32", 6, 2, 256),
          ("f16", 40, 2, 64), ("bf16", 51, 3, 128)]


@pytest.mark.parametrize("dt,h,kv,hd", SHAPES)
@pytest.mark.parametrize("bs", [16, 64])
def test_attention_of_single_tokens(gpu, dt, h, kv, hd, bs):
    c = Case(gpu, h + hd + bs, dt, h, kv, hd, bs,
             [1, 0, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 300, 1000])
    out = c.run()
    c.cache.check()
    assert out.dtype == TD[dt]
    c.check(out)
    wide = c.run(out_dtype=torch.float32)
    c.check(wide, "f32")
    # the bounds of the launch do not change what is computed beyond rounding
    c.check(c.run(max_context_len=20000))


@pytest.mark.parametrize("dt,h,kv,hd", SHAPES)
def test_attention_of_chunks(gpu, dt, h, kv, hd):
    c = Case(gpu, 7 * h + hd, dt, h, kv, hd, 16, [5, 40, 1, 200, 77, 33, 0, 0, 130, 3],
             [5, 3, 1, 70, 2, 0, 0, 1, 19, 9])
    out = c.run()
    c.cache.check()
    c.check(out)
    c.check(c.run(max_q_len=300))


@pytest.mark.parametrize("dt,h,kv,hd,bs", [("bf16", 32, 8, 128, 64), ("f16", 32, 4, 64, 256),
                                           ("f16", 16, 8, 256, 32), ("bf16", 14, 2, 64, 128),
                                           ("f32", 32, 8, 128, 256), ("bf16", 200, 1, 64, 16)])
def test_attention_of_chunks_in_blocks(gpu, dt, h, kv, hd, bs):
    c = Case(gpu, 8 * h + hd, dt, h, kv, hd, bs, [300, 64, 1, 65, 1500, 0, 33], [40, 64, 1, 9, 33, 0, 33])
    out = c.run()
    c.cache.check()
    c.check(out)


def normal_rows(gpu, dt, h, kv, hd, rows):
    """A sequence of 2000 normal keys and values, its result, and the plain one's."""
    c = Case(gpu, h + hd, dt, h, kv, hd, 16, [2000], [rows])
    k, v = c.rng.normal(size=(2, c.cache.num_blocks * 16, kv, hd))
    k, kx = typed(k.astype(np.float32), dt, gpu)
    v, vx = typed(v.astype(np.float32), dt, gpu)
    c.pool.q4_append(k, v, torch.arange(len(k), dtype=torch.int32, device=gpu))
    c.take(kx, vx)
    want = ref.attention(c.qx, *c.rows(0)[0], rows, c.scale, *c.rows(0)[1])[0]
    return host(c.run(out_dtype=torch.float32)).reshape(want.shape), want


@pytest.mark.parametrize("h,kv,hd,rows", [(32, 8, 64, 1), (32, 8, 128, 1), (16, 8, 256, 1), (32, 8, 128, 9)])
def test_f32_attention_is_f32(gpu, h, kv, hd, rows):
    """Offsets and codes of values cancel, all the more over many keys: what is lost before
    they do shows.  Scores are below 16 here, where half a step is 2^-21; one sums up hd
    products, whose roundings add up at random to 2^-21 sqrt(hd / 3) at most, 2^-17.7
    for 256: weights, and so results in norm, are off by that."""
    got, want = normal_rows(gpu, "f32", h, kv, hd, rows)
    assert np.linalg.norm(got - want) <= 2.0 ** -17.7 * np.linalg.norm(want)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("h,kv,hd,rows", [(32, 8, 64, 1), (32, 8, 128, 1), (16, 8, 256, 1), (32, 8, 128, 3)])
def test_f32_results_of_16_bit_queries(gpu, dt, h, kv, hd, rows):
    """Nothing is rounded to 16 bits but weights, in two parts (2^-22).  The matrix
    instructions keep a product of a code as a subnormal to 2^-13 of the largest of eight
    query elements, 2^-12 here, which takes bits of elements below 1/4, a fifth of them: at random
    2^-12 sqrt(hd / 5 / 12) steps of the keys, of 0.3, times the scale, 2^-16.7 at any
    hd (0.3 2^-12 / sqrt(60)): what weights, and results in norm, are off by."""
    got, want = normal_rows(gpu, dt, h, kv, hd, rows)
    assert np.linalg.norm(got - want) <= 2.0 ** -16 * np.linalg.norm(want)


@pytest.mark.parametrize("dt,h,kv,hd,bs", [("bf16", 32, 8, 128, 16), ("f16", 32, 4, 64, 256),
                                           ("f32", 14, 2, 64, 32), ("bf16", 16, 8, 256, 16)])
def test_attention_of_long_contexts(gpu, dt, h, kv, hd, bs):
    c = Case(gpu, 11, dt, h, kv, hd, bs, [9001, 4096, 70, 2047])
    c.check(c.run())
    c = Case(gpu, 12, dt, h, kv, hd, bs, [5001, 130, 2100], [3, 2, 5])
    c.check(c.run())


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("k_by,v_by,q_by,scale", [(1, 1e-4, 1, None), (1, 2e3, 1, None),
                                                  (8, 1, 8, None), (30, 100, 1, None),
                                                  (1, 1, 1e-3, None), (1e-4, 1, 1, None),
                                                  (1, 1, 1, -0.1), (1, 1, 1, 0.0),
                                                  (1, 1, 100, 1e-4)])
def test_attention_of_large_and_small_values(gpu, dt, k_by, v_by, q_by, scale):
    c = Case(gpu, 13, dt, 8, 2, 64, 16, [1, 33, 700, 2500], k_by=k_by, v_by=v_by, q_by=q_by,
             scale=scale)
    c.check(c.run())


def test_attention_where_scales_of_values_jump(gpu):
    # the first tokens' values are tiny, later ones' large, and the other way round
    for order in (1, -1):
        c = Case(gpu, 14, "bf16", 8, 2, 128, 16, [900, 64])
        n = c.k.shape[0]
        by = np.geomspace(1e-4, 3e3, n)[::order, None, None]
        slot = torch.arange(n, dtype=torch.int32, device=gpu)
        v, vx = typed(c.rng.normal(size=(n, 2, 128)) * by, "bf16", gpu)
        k, kx = typed(c.rng.normal(size=(n, 2, 128)), "bf16", gpu)
        c.pool.q4_append(k, v, slot)
        c.take(kx, vx)
        c.check(c.run())


def test_attention_leaves_rows_alone_and_reports(gpu):
    c = Case(gpu, 15, "f16", 8, 2, 64, 16, [40, 60, 100, 30], [2, 3, 4, 1])
    out = torch.full((14, 8 * 64), 7.0, dtype=torch.float16, device=gpu)
    c.q = torch.cat((c.q, torch.zeros_like(c.q[:4])))
    # the third sequence is longer than the bound, the chunk of the second is
    c.run(out=out, max_context_len=60, max_q_len=2)
    with pytest.raises(pagedkv.PagedKvError, match="context-length"):
        c.cache.check()
    assert torch.all(out[2:9] == 7) and torch.all(out[10:] == 7)
    c.check(out[:10], skip=(1, 2))
    # a block id outside the pool: its keys are not attended
    c = Case(gpu, 16, "bf16", 8, 2, 64, 16, [40, 64])
    c.tables[0, 1] = 10 ** 6
    got = c.run()
    with pytest.raises(pagedkv.PagedKvError, match="block-id"):
        c.cache.check()
    k, v, kt, vt = (np.concatenate((x[c.tables[0, 0] * 16:][:16], x[c.tables[0, 2] * 16:][:8]))
                    for x in (c.k, c.v, *c.terms))
    want, *abc = ref.attention(c.qx[:1], k, v, 1, c.scale, kt, vt)
    tol = ref.tolerance(want, *abc, 40, 64, Q4_WEIGHT, HALF["bf16"])
    assert np.all(np.abs(host(got[:1]).reshape(want.shape) - want) <= tol)
    c.tables[1, :4] = -1
    c.tables[0, :3] = (0, 1, 2)
    got = c.run()
    with pytest.raises(pagedkv.PagedKvError, match="block-id"):
        c.cache.check()
    assert not got[1].any()
    # offsets that run backwards or past the rows
    c = Case(gpu, 17, "f16", 8, 2, 64, 16, [40, 60, 20], [2, 3, 1])
    for cu in ([0, 2, 1, 6], [0, -1, 5, 6], [0, 2, 5, 9]):
        out = torch.full((6, 512), 7.0, dtype=torch.float16, device=gpu)
        c.pool.q4_attention(c.q, i32(c.tables, gpu), i32(c.ctx, gpu), cu_q_lens=i32(cu, gpu),
                            max_q_len=4, out=out)
        with pytest.raises(pagedkv.PagedKvError, match="context-length"):
            c.cache.check()


def test_attention_reads_rows_at_a_stride(gpu):
    c = Case(gpu, 18, "bf16", 8, 2, 128, 16, [50, 3, 200])
    wide = torch.randn((3, 20, 128), device=gpu).to(torch.bfloat16)
    wide[:, 4:12] = c.q
    plain = c.run()
    c.q = wide[:, 4:12]
    assert torch.equal(c.run(), plain)


# ---------------------------------------------------------------------------
# packed prompt attention
# ---------------------------------------------------------------------------
def prompt_case(gpu, seed, dt, h, kv, hd, lens, lead=0, tail=0, packed=False, by=1.0):
    rng = np.random.default_rng(seed)
    total = lead + sum(lens) + tail
    x, xx = typed(rng.normal(size=(total, h + 2 * kv, hd)) * by, dt, gpu)
    q, k, v = x.split((h, kv, kv), 1)
    if not packed:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    cu = lead + np.concatenate(([0], np.cumsum(lens)))
    return q, k, v, cu, np.split(xx, (h, h + kv), 1)


def prompt_check(out, cu, xs, dt, scale, out_dt=None):
    q, k, v = xs
    h, hd = q.shape[1:]
    got = host(out).reshape(-1, h, hd)
    for a0, b0 in zip(cu, cu[1:]):
        if b0 <= a0:
            continue
        m = b0 - a0
        want, *abc = ref.attention(q[a0:b0], k[a0:b0], v[a0:b0], m, scale)
        tol = ref.tolerance(want, *abc, m, hd, PROMPT_WEIGHT[dt], HALF[out_dt or dt])
        err = np.abs(got[a0:b0] - want)
        assert np.all(err <= tol), (m, np.unravel_index((err / tol).argmax(), err.shape),
                                    float((err / tol).max()))


@pytest.mark.parametrize("dt,h,kv,hd", SHAPES)
def test_prompts(gpu, dt, h, kv, hd):
    lens = [1, 0, 2, 15, 33, 64, 65, 127, 130]
    q, k, v, cu, xs = prompt_case(gpu, h + hd, dt, h, kv, hd, lens, packed=h % 3 == 2)
    out = pagedkv.prompt_attention(q, k, v, cu.tolist())
    assert out.dtype == TD[dt]
    prompt_check(out, cu, xs, dt, hd ** -0.5)
    wide = pagedkv.prompt_attention(q, k, v, i32(cu, gpu), out_dtype=torch.float32, scale=0.2)
    prompt_check(wide, cu, xs, dt, 0.2, "f32")


@pytest.mark.parametrize("dt,h,kv,hd,lens", [("bf16", 8, 2, 128, [700, 257]), ("f16", 4, 4, 64, [513]),
                                             ("f32", 4, 2, 128, [300]), ("bf16", 4, 2, 256, [400, 3])])
def test_longer_prompts(gpu, dt, h, kv, hd, lens):
    q, k, v, cu, xs = prompt_case(gpu, 21, dt, h, kv, hd, lens, packed=True)
    prompt_check(pagedkv.prompt_attention(q, k, v, i32(cu, gpu), max_len=max(lens)), cu, xs, dt,
                 hd ** -0.5)
    # a bound that is too small costs time only
    prompt_check(pagedkv.prompt_attention(q, k, v, i32(cu, gpu), max_len=1), cu, xs, dt, hd ** -0.5)


@pytest.mark.parametrize("dt,hd", [("f32", 64), ("f32", 128), ("f32", 256), ("f16", 64), ("f16", 256),
                                   ("bf16", 128), ("bf16", 256)])
def test_many_prompts(gpu, dt, hd):
    """More tiles and heads than fill the GPU twice: waves have a unit each."""
    lens = [1, 97, 32, 33, 0, 64, 65, 5] + np.random.default_rng(hd).integers(1, 97, 90).tolist()
    q, k, v, cu, xs = prompt_case(gpu, 25, dt, 14, 2, hd, lens, packed=True)
    prompt_check(pagedkv.prompt_attention(q, k, v, i32(cu, gpu), max_len=97), cu, xs, dt, hd ** -0.5)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("by,scale", [(20.0, 0.125), (1e-3, 0.125), (1.0, -0.3), (1.0, 0.0)])
def test_prompts_of_large_and_small_values(gpu, dt, by, scale):
    q, k, v, cu, xs = prompt_case(gpu, 22, dt, 4, 2, 64, [150, 40], by=by)
    prompt_check(pagedkv.prompt_attention(q, k, v, i32(cu, gpu), scale=scale), cu, xs, dt, scale)


@pytest.mark.parametrize("dt,hd", [("f32", 64), ("f16", 128), ("bf16", 64), ("bf16", 256)])
def test_prompts_see_nothing_outside(gpu, dt, hd):
    lens, lead, tail = [3, 70, 128, 1], 5, 9
    q, k, v, cu, xs = prompt_case(gpu, 23, dt, 4, 2, hd, lens, lead, tail)
    for x in (q, k, v):  # rows of no prompt may hold anything
        x[:lead], x[-tail:] = math.nan, math.inf
    out = torch.full((q.shape[0], 4 * hd), 7.0, dtype=TD[dt], device=gpu)
    pagedkv.prompt_attention(q, k, v, i32(cu, gpu), out=out)
    prompt_check(out, cu, xs, dt, hd ** -0.5)
    assert torch.all(out[:lead] == 7) and torch.all(out[-tail:] == 7)


def test_prompts_with_bad_offsets_are_left_out(gpu):
    q, k, v, cu, xs = prompt_case(gpu, 24, "bf16", 4, 2, 64, [30, 40, 50])
    for cu in ([0, 30, 20, 200], [-4, 30, 70, 120], [0, 30, 70, 121], [130, 140, 20, 2 ** 31 - 1]):
        out = torch.full((120, 256), 7.0, dtype=torch.bfloat16, device=gpu)
        pagedkv.prompt_attention(q, k, v, i32(cu, gpu), max_len=60, out=out)
        seen = np.zeros(120, bool)
        for a, b in zip(cu, cu[1:]):
            if 0 <= a < b <= 120:
                seen[a:b] = True
                prompt_check(out, np.array([a, b]), xs, "bf16", 0.125)
        assert torch.all(out[torch.tensor(~seen)] == 7)
    assert pagedkv.prompt_attention(q, k, v, i32([0], gpu)).shape == (120, 256)
    empty = pagedkv.prompt_attention(q[:0], k[:0], v[:0], i32([0, 0], gpu))
    assert empty.shape == (0, 256)


# ---------------------------------------------------------------------------
# logits
# ---------------------------------------------------------------------------
def logits_case(gpu, seed, dt, b, v, hist, bias, masks):
    rng = np.random.default_rng(seed)
    x, xx = typed(rng.normal(size=(b, v)) * 4, dt, gpu)
    x[:, v // 3], xx[:, v // 3] = -math.inf, -math.inf
    n = rng.integers(0, hist + 1, b)
    m = rng.integers(0, bias + 1, b)
    d = dict(
        tokens=rng.integers(-2, min(v, 40) + 2, n.sum()), cu_tokens=np.concatenate(([0], np.cumsum(n))),
        prompt_lens=rng.integers(0, hist + 1, b), repetition=rng.uniform(0.5, 2.0, b),
        presence=rng.normal(size=b), frequency=rng.normal(size=b),
        bias_tokens=rng.integers(-2, v + 2, m.sum()), bias_values=rng.normal(size=m.sum()) * 9,
        cu_bias=np.concatenate(([0], np.cumsum(m))))
    d["repetition"][::4] = 1.0
    if masks:
        d["mask"] = rng.integers(-2 ** 31, 2 ** 31, (masks, (v + 31) // 32 + seed % 2))
        d["mask_rows"] = rng.integers(-1, masks + 1, b)
    return x, xx, d


def on(d, gpu):
    f = ("repetition", "presence", "frequency", "bias_values")
    return {k: torch.tensor(v, dtype=torch.float32 if k in f else torch.int32, device=gpu)
            for k, v in d.items()}


def logits_want(xx, d):
    out = np.empty(xx.shape, np.float32)
    for b in range(len(xx)):
        a, z = d["cu_tokens"][b:b + 2] if "cu_tokens" in d else (0, 0)
        ba, bz = d["cu_bias"][b:b + 2] if "cu_bias" in d else (0, 0)
        row = -1 if "mask" not in d else d["mask_rows"][b] if "mask_rows" in d else b
        get = lambda k, other: np.float32(d[k][b]) if k in d else np.float32(other)  # noqa: E731
        out[b] = ref.adjust_logits(
            xx[b], d["tokens"][a:z] if "tokens" in d else [], None,
            int(d["prompt_lens"][b]) if "prompt_lens" in d else 0, get("repetition", 1),
            get("presence", 0), get("frequency", 0),
            list(zip(d["bias_tokens"][ba:bz], np.float32(d["bias_values"][ba:bz])))
            if "cu_bias" in d else [],
            d["mask"][row] if 0 <= row < len(d.get("mask", ())) else None,
            "mask" in d and row >= len(d["mask"]))
    return out


def same(got, want, dt):
    w = torch.tensor(want).to(TD[dt])
    return torch.equal(got.cpu().view(torch.int16 if dt != "f32" else torch.int32),
                       w.view(torch.int16 if dt != "f32" else torch.int32))


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("b,v,hist,bias,masks", [(1, 1, 3, 2, 1), (5, 33, 60, 9, 2), (7, 1000, 300, 40, 3),
                                                 (3, 9001, 5, 0, 0), (4, 32000, 900, 70, 2),
                                                 (2, 128256, 2000, 5, 1)])
def test_logits(gpu, dt, b, v, hist, bias, masks):
    x, xx, d = logits_case(gpu, b + v, dt, b, v, hist, bias, masks)
    want = logits_want(xx, d)
    assert same(pagedkv.adjust_logits(x, **on(d, gpu)), want, dt)
    # at odd strides and places, into such ones
    wide = torch.zeros((b, v + 3), dtype=TD[dt], device=gpu)
    wide[:, 1:v + 1] = x
    out = torch.full((b, 2 * v + 5), 7.0, dtype=TD[dt], device=gpu)
    pagedkv.adjust_logits(wide[:, 1:v + 1], **on(d, gpu), out=out[:, v:2 * v])
    assert same(out[:, v:2 * v], want, dt)
    assert torch.all(out[:, :v] == 7) and torch.all(out[:, 2 * v:] == 7)
    # in place, nothing beside the row is touched
    view = wide[:, 1:v + 1]
    assert pagedkv.adjust_logits(view, **on(d, gpu), out=view) is view
    assert same(view, want, dt) and not wide[:, 0].any() and not wide[:, v + 1:].any()


@pytest.mark.parametrize("keep", [(), ("tokens", "cu_tokens"), ("tokens", "cu_tokens", "repetition"),
                                  ("tokens", "cu_tokens", "frequency", "prompt_lens"),
                                  ("tokens", "cu_tokens", "presence"), ("mask", "mask_rows"),
                                  ("bias_tokens", "bias_values", "cu_bias")])
def test_logits_with_parts_left_out(gpu, keep):
    x, xx, d = logits_case(gpu, 5, "f16", 4, 700, 50, 20, 2)
    d = {k: d[k] for k in keep}
    assert same(pagedkv.adjust_logits(x, **on(d, gpu)), logits_want(xx, d), "f16")


def test_logits_odd_arguments(gpu):
    x, xx, d = logits_case(gpu, 6, "f32", 6, 500, 80, 30, 0)
    # penalties that are none, and requests whose offsets run backwards
    d["repetition"][:4] = (0.0, -1.0, np.inf, np.nan)
    assert same(pagedkv.adjust_logits(x, **on(d, gpu)), logits_want(xx, d), "f32")
    t = on(d, gpu)
    t["cu_tokens"] = i32([10, 5, -3, 2 ** 31 - 1, 7, 7, 3], gpu)
    t["cu_bias"] = i32([0, 0, 0, 0, 9, 1 << 30, 4], gpu)
    n, m = len(d["tokens"]), len(d["bias_tokens"])
    got = pagedkv.adjust_logits(x, **t)
    for b, (a, z, ba, bz, first) in enumerate([(0, 0, 0, 0, 0), (0, 0, 0, 0, 0), (0, n, 0, 0, -3),
                                               (0, 0, 0, 9, 0), (7, 7, 9, m, 7), (0, 0, 0, 0, 0)]):
        e = dict(d, tokens=d["tokens"][a:z], cu_tokens=[0, max(z - a, 0)],
                 bias_tokens=d["bias_tokens"][ba:bz], bias_values=d["bias_values"][ba:bz],
                 cu_bias=[0, max(bz - ba, 0)])
        for k in ("repetition", "presence", "frequency", "prompt_lens"):
            e[k] = d[k][b:b + 1]
        if b == 2:
            e["prompt_lens"] = np.maximum(d["prompt_lens"][b:b + 1] - 3, 0)
        assert same(got[b:b + 1], logits_want(xx[b:b + 1], e), "f32"), b
    # NaN stays where it is allowed, the mask row of a request is its own without mask_rows
    x[0, 5] = math.nan
    mask = torch.zeros((6, 16), dtype=torch.int32, device=gpu)
    mask[0, 0] = 0b110000
    got = pagedkv.adjust_logits(x, mask=mask)
    assert torch.isnan(got[0, 5]) and got[0, 4] == x[0, 4]
    assert torch.all(got[1:] == -math.inf) and torch.all(got[0, 6:] == -math.inf)
    assert pagedkv.adjust_logits(x[:0]).shape == (0, 500)


# ---------------------------------------------------------------------------
# together: streams, graphs, a run of them
# ---------------------------------------------------------------------------
def test_on_another_stream(gpu):
    c = Case(gpu, 31, "bf16", 8, 2, 128, 16, [50, 3, 2000])
    plain = c.run()
    q, k, v, cu, xs = prompt_case(gpu, 32, "bf16", 8, 2, 128, [100, 20])
    prompt = pagedkv.prompt_attention(q, k, v, i32(cu, gpu))
    x, xx, d = logits_case(gpu, 33, "f16", 4, 700, 50, 20, 2)
    d = on(d, gpu)
    logits = pagedkv.adjust_logits(x, **d)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    slots = i32(np.arange(48), gpu)
    # inputs made on the current stream just before
    k2, v2 = (torch.randn((48, 2, 128), device=gpu).to(torch.bfloat16) for _ in range(2))
    c.pool.q4_append(k2, v2, slots, stream=side)
    kk, _ = c.pool.q4_gather(slots, stream=side)
    side.synchronize()
    assert np.array_equal(host(kk), ref.held(host(k2)).astype(np.float32))
    c2 = Case(gpu, 31, "bf16", 8, 2, 128, 16, [50, 3, 2000])
    a = c2.run(stream=side)
    b = pagedkv.prompt_attention(q + 0, k + 0, v + 0, i32(cu, gpu), stream=side)
    e = pagedkv.adjust_logits(x + 0, **d, stream=side)
    side.synchronize()
    assert torch.equal(a, plain) and torch.equal(b, prompt) and torch.equal(e, logits)


def serving_step(pool, t, layers=1):
    """Prompts and decodes of one step; everything is on the device."""
    o = pagedkv.prompt_attention(t["pq"], t["pk"], t["pv"], t["cu"], max_len=64)
    pool.q4_append(t["pk"], t["pv"], t["p_slots"])
    pool.q4_append(t["dk"], t["dv"], t["d_slots"])
    a = pool.q4_attention(t["dq"], t["tables"], t["ctx"], max_context_len=96)
    x = a.float() @ t["w"]
    x = pagedkv.adjust_logits(x, tokens=t["tokens"], cu_tokens=t["cu_tokens"],
                              repetition=t["rep"], mask=t["mask"], mask_rows=t["rows"], out=x)
    return o, a, x


def step_inputs(gpu, seed, kv=2, h=8, hd=64, bs=16):
    g = torch.Generator(device=gpu).manual_seed(seed)

    def r(*shape):
        return torch.randn(shape, generator=g, device=gpu).to(torch.bfloat16)

    t = dict(pq=r(70, h, hd), pk=r(70, kv, hd), pv=r(70, kv, hd), cu=i32([0, 40, 70], gpu),
             dq=r(3, h, hd), dk=r(3, kv, hd), dv=r(3, kv, hd))
    # two prompts of 40 and 30 tokens in blocks 0-2 and 3-4, then a token more each; a third one
    t["p_slots"] = i32(list(range(40)) + [48 + i for i in range(30)], gpu)
    t["tables"] = i32([[0, 1, 2], [3, 4, 0], [5, 0, 0]], gpu)
    t["d_slots"] = i32([40, 78, 80], gpu)
    t["ctx"] = i32([41, 31, 1], gpu)
    t["w"] = torch.randn((h * hd, 300), generator=g, device=gpu)
    t["tokens"], t["cu_tokens"] = i32([5, 5, 9, 200], gpu), i32([0, 2, 4, 4], gpu)
    t["rep"] = torch.tensor([1.3, 0.8, 2.0], device=gpu)
    t["mask"] = torch.randint(-2 ** 31, 2 ** 31, (1, 10), generator=g, device=gpu).int()
    t["rows"] = i32([0, -1, 0], gpu)
    return t


def test_a_step_of_them_together(gpu):
    t = step_inputs(gpu, 1)
    cache = pagedkv.PagedKvCache(1, 6, 16, 2, 64, pagedkv.Q4)
    o, a, x = serving_step(cache.layer(0), t)
    cache.check()
    prompt_check(o, np.array([0, 40, 70]), [host(t[n]) for n in ("pq", "pk", "pv")], "bf16", 0.125)
    pk, pv, dk, dv, dq = (host(t[n]) for n in ("pk", "pv", "dk", "dv", "dq"))
    for i, (lo, hi) in enumerate([(0, 40), (40, 70), (0, 0)]):
        k, v = np.concatenate((pk[lo:hi], dk[i:i + 1])), np.concatenate((pv[lo:hi], dv[i:i + 1]))
        want, *abc = ref.attention(dq[i:i + 1], ref.held(k), ref.held(v), 1, 0.125,
                                    ref.held_terms(k), ref.held_terms(v))
        tol = ref.tolerance(want, *abc, len(k), 64, Q4_WEIGHT, HALF["bf16"])
        assert np.all(np.abs(host(a[i:i + 1]).reshape(want.shape) - want) <= tol)
    y = (a.float() @ t["w"]).cpu().numpy()
    for i, toks in enumerate(([5, 5], [9, 200], [])):
        want = ref.adjust_logits(y[i], toks, None, 0, np.float32([1.3, 0.8, 2.0][i]), 0, 0, [],
                                 None if i == 1 else t["mask"][0].cpu().numpy())
        assert np.array_equal(x[i].cpu().numpy(), want)
    tokens = pagedkv.sample(x, torch.tensor([0.0, 0.7, 0.0], device=gpu))
    assert tokens[0] == x[0].argmax() and tokens[2] == x[2].argmax()


def test_captured_steps_replay(gpu):
    # two graphs of one step over two pools, replayed in turn beside eager work
    graphs = []
    for seed in (1, 2):
        t = step_inputs(gpu, seed)
        cache = pagedkv.PagedKvCache(1, 6, 16, 2, 64, pagedkv.Q4)
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            serving_step(cache.layer(0), t)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = serving_step(cache.layer(0), t)
        graphs.append((t, cache, g, out))
    for round_ in range(3):
        for seed, (t, cache, g, out) in enumerate(graphs):
            fresh = step_inputs(gpu, 10 * round_ + seed)
            for n in t:
                t[n].copy_(fresh[n])
            want_cache = pagedkv.PagedKvCache(1, 6, 16, 2, 64, pagedkv.Q4)
            g.replay()
            want = serving_step(want_cache.layer(0), fresh)
            torch.cuda.synchronize()
            for got, w in zip(out, want):
                assert torch.equal(got.view(torch.uint8), w.view(torch.uint8))
            cache.check()
            want_cache.close()


def test_a_captured_decode_follows_lengths(gpu):
    # the same graph serves growing contexts: split work is joined from device lengths
    c = Case(gpu, 34, "bf16", 32, 8, 128, 16, [3000, 700, 1])
    cl, tables = i32(c.ctx, gpu), i32(c.tables, gpu)
    kw = dict(max_context_len=3000, scale=c.scale)
    c.pool.q4_attention(c.q, tables, cl, **kw)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = c.pool.q4_attention(c.q, tables, cl, **kw)
    for ctx in ([3000, 700, 1], [5, 690, 0], [2999, 1, 1], [3000, 700, 1]):
        cl.copy_(i32(ctx, gpu))
        c.ctx = ctx
        g.replay()
        eager = c.pool.q4_attention(c.q, tables, cl, **kw)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        c.check(out)


def test_two_calls_at_once_have_scratch_of_their_own(gpu):
    c = Case(gpu, 35, "f16", 32, 8, 64, 16, [4000, 2500])
    d = Case(gpu, 36, "f16", 32, 8, 64, 16, [3900, 100])
    want = c.run(), d.run()
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(4):
        got = [x.run(stream=s) for x, s in zip((c, d), streams)]
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_other_calls_refuse_a_pool_of_4_bits(gpu):
    cache = pagedkv.PagedKvCache(1, 4, 16, 2, 64, pagedkv.Q4)
    L, h = pagedkv.lib(), cache.handle
    t = torch.zeros(4096, device=gpu)
    p = t.data_ptr()
    calls = {
        "pkv_append": (h, 0, p, p, p, 1, None),
        "pkv_gather_seq": (h, 0, p, 1, p, p, None),
        "pkv_gather_varlen": (h, 0, p, 1, p, 1, 1, p, p, None),
        "pkv_decode_attention": (h, 0, p, p, 0, p, 1, p, 1, 1, 4, 0.1, None, None, None),
        "pkv_decode_attention_noalloc": (h, 0, p, p, 0, p, 1, p, 1, 1, 4, 0.1, None, None, None),
        "pkv_decode_attention_positions": (h, 0, p, p, 0, p, 1, p, p, 1, 1, 4, 0.1, None, None, None),
        "pkv_prefill_attention": (h, 0, p, p, 0, p, p, p, 1, 1, 1, 1, 4, 0.1, None),
        "pkv_mixed_attention": (h, 0, None, None, 4, 0.1, None),
        "pkv_pool_reserve_decode": (h, 1, 4, 16),
        "pkv_pool_reserve_prefill": (h, 1, 4, 16, 16),
        "pkv_pool_fill_normal": (h, 1, None),
        "pkv_key_bounds": (h, 0, p, p, 1, None, p, 1, 1, None),
        "pkv_select_blocks": (h, p, p, p, 2, 1, 1, None, p, p, 1, 1, 1, 1, 16, 4, p, 1 << 14, None),
        "pkv_sparse_attention": (h, 0, p, p, 0, p, 1, None, p, p, 1, 1, 1, 1, 4, 0.1, p, 1 << 14, None),
    }
    for name, args in calls.items():
        assert getattr(L, name)(*args) == -4, name
        assert b"PKV_Q4" in L.pkv_last_error(h), name
    assert L.pkv_decode_workspace_bytes(h, 1, 4, 100) == 0
    assert L.pkv_key_bounds_bytes(h) == 0
    plain = pagedkv.PagedKvCache(1, 4, 16, 2, 64, torch.float16)
    for name, args in {"pkv_q4_append": (0, p, p, 1, 128, 128, p, 1, None),
                       "pkv_q4_gather": (0, p, 1, p, p, 1, None),
                       "pkv_q4_attention": (0, p, 1, 256, p, 1, None, p, p, 1, 1, 1, 1, 16, 4, 0.1,
                                            None, 0, None)}.items():
        assert getattr(L, name)(plain.handle, *args) == -4, name
    with pytest.raises(TypeError, match="Q4"):
        plain.layer(0).q4_gather(i32([0], gpu))
    with pytest.raises(pagedkv.PagedKvError, match="at least 16"):
        pagedkv.PagedKvCache(1, 4, 8, 2, 64, pagedkv.Q4)
    torch.cuda.synchronize()
    assert not t.any()


def test_refusals_of_the_pool_calls(gpu):
    cache = pagedkv.PagedKvCache(1, 4, 16, 2, 64, pagedkv.Q4)
    L, h = pagedkv.lib(), cache.handle
    x = torch.zeros(1 << 16, device=gpu)
    p = x.data_ptr()

    def append(k=p, v=p, dt=1, ks=128, vs=128, slots=p, n=2, layer=0):
        return L.pkv_q4_append(h, layer, k, v, dt, ks, vs, slots, n, None)

    for bad in (dict(layer=1), dict(n=-1), dict(dt=3), dict(k=None), dict(v=p + 2), dict(slots=p + 1),
                dict(ks=127), dict(ks=132), dict(vs=64), dict(slots=None), dict(ks=1 << 62)):
        assert append(**bad) == -1, bad
    assert append(n=0, k=None) == 0

    def gather(slots=p, n=2, k=p, v=p, dt=0):
        return L.pkv_q4_gather(h, 0, slots, n, k, v, dt, None)

    for bad in (dict(slots=None), dict(n=-1), dict(k=p + 4), dict(dt=3), dict(v=None)):
        assert gather(**bad) == -1, bad
    far = p + (1 << 17)

    def attend(q=p, qdt=1, qs=256, out=far, odt=1, cu=None, cl=p, bt=p, mb=1, n=2, rows=2, mq=1, mc=16,
               nh=4, scale=0.1, ws=None, wb=0):
        return L.pkv_q4_attention(h, 0, q, qdt, qs, out, odt, cu, cl, bt, mb, n, rows, mq, mc, nh,
                                  scale, ws, wb, None)

    for bad in (dict(q=None), dict(out=None), dict(cl=None), dict(bt=None), dict(q=p + 8), dict(qdt=3),
                dict(odt=2), dict(qs=255), dict(qs=260), dict(mb=0), dict(n=-1), dict(rows=3),
                dict(mq=2), dict(mq=0), dict(mc=0), dict(mc=(1 << 30) + 1), dict(nh=3), dict(nh=0),
                dict(scale=math.nan), dict(scale=math.inf), dict(out=p + 16), dict(cl=p + 2)):
        assert attend(**bad) == -1, bad
    need = L.pkv_q4_workspace_bytes(h, 2, 2, 1, 1 << 20, 4)
    if need:
        assert attend(mc=1 << 20) == -1 and attend(mc=1 << 20, ws=far + (1 << 18), wb=need - 1) == -1
    assert attend(n=0, rows=0, q=None) == 0
    assert L.pkv_q4_workspace_bytes(h, 2, 2, 1, 16, 3) == 0
    torch.cuda.synchronize()
    assert not x.any()
