"""Plain 64-bit implementations of serving from a cache held in 4 bits (rows into a
pool and back, attention over it, packed prompt attention, adjusted logits),
written from their definitions.  Only the tests use them."""
import numpy as np

GROUP = 32
LIMIT = 65024.0  # m + 15 s stays in the f16 range


def f16(x):
    """Nearest f16, as float64."""
    with np.errstate(over="ignore"):
        return np.asarray(x, np.float32).astype(np.float16).astype(np.float64)


def quantize(x):
    """(codes, m, s) of rows x (..., hd): codes as x, m and s (..., hd / 32)."""
    x = np.asarray(x, np.float64)
    x = np.clip(np.where(np.isnan(x), 0.0, x), -LIMIT, LIMIT)
    y = x.reshape(*x.shape[:-1], -1, GROUP)
    m = f16(y.min(-1))
    top = y.max(-1).astype(np.float32)
    s = f16((top - m.astype(np.float32)) / np.float32(15.0))
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.rint((y - m[..., None]) / s[..., None])
    c = np.where(s[..., None] > 0, np.clip(c, 0, 15), 0)
    return c.reshape(x.shape).astype(np.int64), m, s


def stands_for(c, m, s):
    y = c.reshape(*c.shape[:-1], -1, GROUP)
    return (m[..., None] + s[..., None] * y).reshape(c.shape)


def held(x):
    return stands_for(*quantize(x))


def held_terms(x):
    """|m| + s c of x's elements: the two terms that an element's value is the sum of."""
    c, m, s = quantize(x)
    return stands_for(c, np.abs(m), s)


def chunk_bytes(k, c, m, s, bs):
    """Bytes of one block and kv head, from codes (bs, hd), m, s (bs, G); k: keys."""
    hd = c.shape[1]
    g, t = hd // 32, hd // 16
    words = np.zeros(0, np.uint8)
    if k:
        w = np.zeros((bs, 4, g), np.uint64)
        for i in range(4):
            for e in range(8):
                bit = 4 * (e // 2 + 4 * (e % 2))
                for j in range(g):
                    w[:, i, j] |= c[:, 32 * j + 8 * i + e].astype(np.uint64) << np.uint64(bit)
        words = w.astype(np.uint32).reshape(-1).view(np.uint8)
    else:
        w = np.zeros((16, bs, t // 2), np.uint8)
        for i in range(16):
            for j in range(t):
                w[i, :, j // 2] |= (c[:, i + 16 * j] << (4 * (j % 2))).astype(np.uint8)
        words = w.reshape(16, bs // 4, 4, t // 2).transpose(1, 0, 2, 3).reshape(-1)

    def quads(x):
        return x.reshape(bs // 4, 4, g).transpose(0, 2, 1).astype(np.float16).reshape(-1).view(np.uint8)

    return np.concatenate((words, quads(s), quads(m)))


def attention(q, keys, values, n_rows, scale, key_terms=None, value_terms=None):
    """Rows q (m, H, hd), the last m of n tokens with keys, values (n, kv, hd): (out,
    A, B, C): the result, sum_k p |v|, the largest sum_d |q| |k| of the row and the
    root of the largest sum_d (q k)^2, from which bounds are made; key_terms,
    value_terms: in the place of |k| and |v| in A and B where these are added up from
    terms that may cancel."""
    key_terms = np.abs(keys) if key_terms is None else key_terms
    value_terms = np.abs(values) if value_terms is None else value_terms
    m, h, hd = q.shape
    n, kv, _ = keys.shape
    out, a = np.zeros((m, h, hd)), np.zeros((m, h, hd))
    b, c = np.zeros((2, m, h))
    for i in range(m):
        seen = n - m + i + 1
        if seen <= 0:
            continue
        for j in range(h):
            kk, vv = keys[:seen, j * kv // h], values[:seen, j * kv // h]
            x = scale * (kk @ q[i, j])
            w = np.exp(x - x.max())
            w /= w.sum()
            out[i, j], a[i, j] = w @ vv, w @ value_terms[:seen, j * kv // h]
            b[i, j] = abs(scale) * (key_terms[:seen, j * kv // h] @ np.abs(q[i, j])).max()
            c[i, j] = abs(scale) * np.sqrt((kk ** 2 @ q[i, j] ** 2).max())
    return out, a, b, c


def tolerance(out, a, b, c, n, hd, weight_step, out_step, key_step=0.0, value_step=0.0):
    """Largest error of attention whose scores and sums are held in f32.

    A score is off by at most (hd + 16) 2^-23 of sum |q| |k| (a product and a sum
    each rounded, the sums in any order and perhaps truncated), and its exponent's
    argument and the exponential by 2^-20 more; two of them enter a weight (its
    own and the denominator's).  Keys that are rounded first, by key_step (half a step)
    each and independently, move a score by key_step / sqrt(3) of the root of sum
    (q k)^2 as a standard deviation, of which six are allowed (exceeded once in 5e8).
    A weight rounded before its product is off by weight_step, a value by value_step, sums
    over n keys by n 2^-23; the result is rounded once, by out_step (half a step
    of its type)."""
    ds = (hd + 16) * 2.0 ** -23 * b[..., None] + 2.0 ** -20
    ds = ds + 6 * key_step / np.sqrt(3.0) * c[..., None]
    rel = np.expm1(2 * ds) + weight_step + value_step + (n + 64) * 2.0 ** -23
    return a * rel * (1 + out_step) + np.abs(out) * out_step + 2.0 ** -24


def adjust_logits(x, tokens, cu, prompt, rep, pres, freq, bias, mask_row, none=False):
    """One row in f32, each operation rounded.  tokens: the request's; prompt: how many
    of them are; bias: list of (token, value); mask_row: words or None."""
    f = np.float32
    x = x.astype(f).copy()
    v = len(x)
    with np.errstate(invalid="ignore", over="ignore"):
        r = f(rep) if rep > 0 and np.isfinite(rep) else f(1)
        for t in {int(t) for t in tokens if 0 <= t < v}:
            x[t] = x[t] / r if x[t] > 0 else x[t] * r
            n = sum(1 for u in tokens[max(prompt, 0):] if u == t)
            if n:
                x[t] = f(x[t] - f(f(freq) * f(n)))
                x[t] = f(x[t] - f(pres))
        for t, val in {int(t): val for t, val in bias if 0 <= t < v}.items():
            x[t] = f(x[t] + f(val))
    if none:
        x[:] = -np.inf
    elif mask_row is not None:
        w = np.asarray(mask_row).astype(np.int64) & 0xffffffff
        t = np.arange(v)
        x[((w[t // 32] >> (t % 32)) & 1) == 0] = -np.inf
    return x
